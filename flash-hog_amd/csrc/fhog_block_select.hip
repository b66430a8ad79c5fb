// Which blocks of a paged cache a new token attends to (fhog_blocks.h).
//
// A full page has the mean of its keys, m_j = sum over its rows / page_size, summed in 64 bits and rounded to
// fp32 once. The sum is exact for fp16 and wherever the values lie within 2^40 or so of each other; beyond that it is a fixed
// order of the rows that makes a mean the same at every call. For a token and key/value head,
// s_j = <sum over its group's queries, m_j> in 64 bits, since a choice has no tolerance: fp32 would choose otherwise
// wherever two scores are within its rounding. The three kernels below add the products in orders of their own, so scores
// within a rounding of 64 bits may be ranked differently by another of them; equal means have equal scores in each. A token at
// position p of pages 0 to p / page_size takes the first `first` and the last `last` of them, and of those
// between the ones with the largest scores, ties to the lowest index; NaN is below every number.
//
// Scores are kept as their bits in an order that compares as they do. Where sequences have many new tokens, 16 of
// them share the means' reads, as matrix products of 64 bits, whose scores stay in LDS, where a wave chooses for a
// token; few tokens have a workgroup each. Else, and for tables wider than LDS, scores go through memory.
#include "fhog_blocks.h"

namespace fhog {

namespace {

constexpr int kThreads = 256;

// Four e4m3 values times their row's scale (e8m0: 0 is 2^-127, 255 NaN), in fp32, exact.
__device__ __forceinline__ f32x4 dequantise4_fp32(uint32_t x, uint32_t code) {
  const float scale = __builtin_bit_cast(float, code == 0 ? 0x00400000u : code == 255 ? 0x7fc00000u : code << 23);
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, true);
  return f32x4{a[0] * scale, a[1] * scale, b[0] * scale, b[1] * scale};
}

// The means of the pages that the new tokens fill. A sequence's new tokens fill at most count / page_size + 1
// pages, so its pages' slots start at offset / page_size + index; a workgroup takes every gridDim-th
// slot and key/value head.
template <typename C, int D> __global__ void __launch_bounds__(kThreads) key_means_kernel(KeyMeansParams<C> p) {
  constexpr int kLanes = D / 8, kRows = kThreads / kLanes;
  __shared__ double box[kRows][D];
  const CacheShape& c = p.at;
  auto first_slot = [&](int b) { return (packed_begin(c, b) >> c.page_shift) + b; };
  const long slots = c.offsets ? (long)first_slot(c.batch) : c.batch;
  const int col = 8 * (int)(threadIdx.x % kLanes), way = threadIdx.x / kLanes;
  for (long i = blockIdx.x; i < slots * c.kv_heads; i += gridDim.x) {
    const int slot = (int)(i / c.kv_heads), hk = (int)(i % c.kv_heads);
    const int b = c.offsets ? last_at_or_before(c.batch, slot, first_slot) : slot;
    const int count = c.offsets ? max(0, packed_begin(c, b + 1) - packed_begin(c, b)) : 1;
    const int length = max(0, c.lengths[b]), before = max(0, length - count);
    const long at = (before >> c.page_shift) + (long)slot - (c.offsets ? first_slot(b) : slot);
    if (at < 0 || at >= length >> c.page_shift || at >= c.pages_per_seq) continue;
    const int page = c.table[(long)b * c.pages_per_seq + at];
    if ((unsigned)page >= (unsigned)c.pages) continue;
    const long line0 = ((long)page * c.kv_heads + hk) << c.page_shift;
    double sum[8] = {};
    for (int r = way; r < 1 << c.page_shift; r += kRows) {
      const C* row = p.k + (line0 + r) * D + col;
      if constexpr (sizeof(C) == 1) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(row);
        const uint32_t code = p.k_scale[line0 + r];
        const f32x4 lo = dequantise4_fp32(x[0], code), hi = dequantise4_fp32(x[1], code);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += (double)lo[e], sum[4 + e] += (double)hi[e];
      } else {
        const V8<C> x = *reinterpret_cast<const V8<C>*>(row);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += (double)(float)x[e];
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) box[way][col + e] = sum[e];
    __syncthreads();
    const int ways = min(kRows, 1 << c.page_shift);
    if ((int)threadIdx.x < D) {
      double total = 0.;
      for (int w = 0; w < ways; ++w) total += box[w][threadIdx.x];
      p.means[((long)page * c.kv_heads + hk) * D + threadIdx.x] = (float)(total / (double)(1 << c.page_shift));
    }
  }
}

// The columns that a token may choose from.
struct TokenBlocks {
  int own;     // its own column, -1 if it sees nothing
  int lo, hi;  // columns [lo, hi) are chosen from by score
  int room;    // how many of them
  // Of a position; most: as if its own column were the table's last at most (no token before it then chooses from more).
  template <typename P> __device__ __forceinline__ TokenBlocks(const P& p, long pos, bool most = false) {
    const long at = pos < 0 ? -1 : pos >> p.at.page_shift;
    own = at < p.at.pages_per_seq ? (int)at : most ? p.at.pages_per_seq - 1 : -1;  // (a length beyond the table)
    lo = min(p.first, own + 1);
    hi = max(lo, own + 1 - p.last);
    room = max(0, p.blocks - lo - (own + 1 - hi));
  }
  __device__ __forceinline__ bool by_score() const { return hi - lo > room; }
};

// A packed token's sequence and position, below 0 if it is of none.
struct TokenAt {
  int b;
  long pos;
  __device__ __forceinline__ TokenAt(const CacheShape& c, int t) {
    b = c.offsets ? last_at_or_before(c.batch, t, [&](int s) { return packed_begin(c, s); }) : t;
    const int begin = packed_begin(c, b), end = c.offsets ? packed_begin(c, b + 1) : b + 1;
    pos = t < begin || t >= end ? -1 : (long)max(0, c.lengths[b]) - (end - t);
  }
};

// A score's bits in an order that compares as scores do, NaN lowest.
__device__ __forceinline__ unsigned long sortable(double x) {
  if (!(x == x)) return 0;
  const long bits = __builtin_bit_cast(long, x + 0.);  // (-0 + 0 = 0)
  return (unsigned long)bits ^ (bits < 0 ? ~0ul : 1ul << 63);
}

// The columns that are not chosen by score, and what is behind the last one, of a token's list; by `threads`
// threads.
__device__ __forceinline__ void write_forced(const TokenBlocks& tb, int* out, int blocks, int thread, int threads) {
  const int count = min(blocks, tb.own + 1);
  const bool by_score = tb.by_score();
  for (int i = thread; i < blocks; i += threads)
    if (!by_score || i < tb.lo || i >= tb.lo + tb.room)
      // (the last ones end with the token's own)
      out[i] = i >= count ? -1 : i < tb.lo || !by_score ? i : tb.own + 1 - (count - i);
}

// The largest value of 32 bits that `want` keys reach, bit by bit from bit `top` of `prefix` on, where count_from
// says how many reach a value; or, sooner, one that exactly `want` reach (exact).
template <typename F> __device__ __forceinline__ uint32_t reached_by(int want, uint32_t prefix, int top, bool& exact, F&& count_from) {
  exact = false;
  for (int bit = top; bit >= 0 && !exact; --bit) {
    const uint32_t next = prefix | 1u << bit;
    const int count = count_from(next);
    if (count >= want) {
      prefix = next;
      exact = count == want;
    }
  }
  return prefix;
}

// The score that sortable() made a key of.
__device__ __forceinline__ double score_of(unsigned long key) {
  return __builtin_bit_cast(double, key >> 63 ? key ^ 1ul << 63 : ~key);
}

// The least and the largest of a wave's lanes, in every lane.
template <typename F> __device__ __forceinline__ float wave_reduce(float x, F&& f) {
  auto step = [&](auto moved) { x = f(x, __builtin_bit_cast(float, moved(__builtin_bit_cast(int, x)))); };
  // (lanes that get nothing keep their own)
  step([](int i) { return __builtin_amdgcn_update_dpp(i, i, 0x111, 0xf, 0xf, false); });  // row_shr:1
  step([](int i) { return __builtin_amdgcn_update_dpp(i, i, 0x112, 0xf, 0xf, false); });
  step([](int i) { return __builtin_amdgcn_update_dpp(i, i, 0x114, 0xf, 0xf, false); });
  step([](int i) { return __builtin_amdgcn_update_dpp(i, i, 0x118, 0xf, 0xf, false); });
  step([](int i) { return __builtin_amdgcn_update_dpp(i, i, 0x142, 0xa, 0xf, false); });  // row_bcast:15
  step([](int i) { return __builtin_amdgcn_update_dpp(i, i, 0x143, 0xc, 0xf, false); });  // row_bcast:31
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

// The `room` largest of a wave's n > room keys, KJ a lane: key j of lane l is column lo + 64 j + l. Writes their
// columns, rising, to out.
// Scores rounded to fp32 keep their order, so a value that exactly `room` of them reach tells the choice; halving
// the range of the scores finds one as soon as it falls between the last one taken and the first one left: seven
// or eight steps for 250 scores, where the bits of the keys, which spend the first dozen on sign and exponent,
// take sixteen to twenty. Equal fp32 scores there, or ones that are not finite, leave it to the keys themselves.
template <int KJ, typename F> __device__ __forceinline__ void choose_in_wave(int n, int lo, int room, int* out, F&& key_of) {
  const int lane = threadIdx.x & 63;
  const unsigned long below = (1ul << lane) - 1;
  int at = 0;
  auto put = [&](int j, bool take) {
    const unsigned long takes = __ballot(take);
    if (take) out[at + __popcll(takes & below)] = lo + 64 * j + lane;
    at += __popcll(takes);
  };
  auto count = [&](auto&& which) {
    int sum = 0;
    if constexpr (KJ <= 4) {
#pragma unroll
      for (int j = 0; j < KJ; ++j) sum += __popcll(__ballot(which(j)));
      return sum;
    } else {  // (a lane's own first: a ballot takes as long as four comparisons)
#pragma unroll
      for (int j = 0; j < KJ; ++j) sum += which(j) ? 1 : 0;
      return wave_sum(sum);
    }
  };
  float f[KJ], least = INFINITY, most = -INFINITY;
  bool good = true;
#pragma unroll
  for (int j = 0; j < KJ; ++j) {  // (not in a branch a key: it would wait for each in turn)
    const float x = (float)score_of(key_of(min(64 * j + lane, n - 1)));
    good = good && fabsf(x) < INFINITY;
    least = fminf(least, x), most = fmaxf(most, x);
    f[j] = 64 * j + lane < n ? x : -INFINITY;
  }
  if (__all(good)) {
    least = wave_reduce(least, [](float a, float b) { return fminf(a, b); });
    most = wave_reduce(most, [](float a, float b) { return fmaxf(a, b); });
    // (all reach `least`; what is reached by too few is above)
    float above = most, middle = 0.5f * least + 0.5f * most;
    while (middle > least && middle <= above) {
      const int reach = count([&](int j) { return f[j] >= middle; });
      if (reach == room) {
#pragma unroll
        for (int j = 0; j < KJ; ++j)
          if (64 * j < n) put(j, f[j] >= middle);
        return;
      }
      if (reach > room)
        least = middle;
      else
        above = middle;
      const float next = 0.5f * least + 0.5f * above;
      if (next == middle) break;
      middle = next;
    }
  }
  uint32_t hi[KJ], low[KJ];  // (0 where there is no key)
  uint32_t any = 0, all = ~0u;
#pragma unroll
  for (int j = 0; j < KJ; ++j) {
    const unsigned long key = key_of(min(64 * j + lane, n - 1));
    const bool there = 64 * j + lane < n;
    hi[j] = there ? (uint32_t)(key >> 32) : 0;
    low[j] = there ? (uint32_t)key : 0;
    any |= hi[j];
    all &= there ? hi[j] : ~0u;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    any |= (uint32_t)__shfl_xor((int)any, d, 64);
    all &= (uint32_t)__shfl_xor((int)all, d, 64);
  }
  any = __builtin_amdgcn_readfirstlane(any), all = __builtin_amdgcn_readfirstlane(all);
  auto there = [&](int j) { return 64 * j + lane < n; };
  const int top = any == all ? -1 : 31 - __builtin_clz(any ^ all);
  const uint32_t same = top < 0 ? ~0u : top == 31 ? 0u : ~((2u << top) - 1);  // bits above that all keys share
  bool exact;
  const uint32_t h = reached_by(room, all & same, top, exact, [&](uint32_t x) { return count([&](int j) { return there(j) && hi[j] >= x; }); });
  uint32_t l = 0;
  int left = 0;  // keys equal to (h, l) that are taken, if not all
  if (!exact) {
    const int more = count([&](int j) { return there(j) && hi[j] > h; });
    l = reached_by(room - more, 0, 31, exact, [&](uint32_t x) { return count([&](int j) { return there(j) && hi[j] == h && low[j] >= x; }); });
    if (!exact) left = room - more - count([&](int j) { return there(j) && hi[j] == h && low[j] > l; });
  }
#pragma unroll
  for (int j = 0; j < KJ; ++j) {
    if (64 * j >= n) continue;
    const bool equal = there(j) && hi[j] == h && low[j] == l;
    bool take = there(j) && (hi[j] > h || (hi[j] == h && low[j] >= l));
    if (!exact) {
      const unsigned long equals = __ballot(equal);
      take = take && (!equal || (int)__popcll(equals & below) < left);
      left = max(0, left - (int)__popcll(equals));
    }
    put(j, take);
  }
}

// ------------------------------------------------------------------ scores

// Sum over sixteen neighbouring lanes, in all of them.
__device__ __forceinline__ double row16_sum(double x) {
  auto step = [&](auto moved) {
    const long bits = __builtin_bit_cast(long, x);
    const uint32_t lo = (uint32_t)moved((int)bits), hi = (uint32_t)moved((int)(bits >> 32));
    x += __builtin_bit_cast(double, (unsigned long)hi << 32 | lo);
  };
  step([](int i) { return __builtin_amdgcn_mov_dpp(i, 0xb1, 0xf, 0xf, true); });   // quad_perm:[1,0,3,2]
  step([](int i) { return __builtin_amdgcn_mov_dpp(i, 0x4e, 0xf, 0xf, true); });   // quad_perm:[2,3,0,1]
  step([](int i) { return __builtin_amdgcn_mov_dpp(i, 0x141, 0xf, 0xf, true); });  // row_half_mirror
  step([](int i) { return __builtin_amdgcn_mov_dpp(i, 0x140, 0xf, 0xf, true); });  // row_mirror
  return x;
}

// A token's scores of kColumns columns for a key/value head; sixteen lanes a column.
constexpr int kColumns = 64;
template <typename T, int D> __global__ void __launch_bounds__(kThreads) block_score_kernel(BlockSelectParams<T> p) {
  constexpr int E = D / 16;
  const CacheShape& c = p.at;
  const int hk = blockIdx.x % c.kv_heads, t = p.token0 + blockIdx.x / c.kv_heads;
  const TokenAt token(c, t);
  const TokenBlocks tb(p, token.pos);
  if (!tb.by_score()) return;
  const int c0 = blockIdx.y * kColumns;
  if (c0 >= tb.hi || c0 + kColumns <= tb.lo) return;
  const int lane = threadIdx.x % 16, way = threadIdx.x / 16, group = p.heads / c.kv_heads;
  double q[E] = {};
  for (int h = 0; h < group; ++h) {
    const T* row = p.q + ((long)t * p.heads + hk * group + h) * D + lane * 4;
#pragma unroll
    for (int j = 0; j < E; j += 4) {
      const V4<T> x = *reinterpret_cast<const V4<T>*>(row + 16 * j);
#pragma unroll
      for (int e = 0; e < 4; ++e) q[j + e] += (double)(float)x[e];
    }
  }
  unsigned long* const scores = p.scores + (long)blockIdx.x * c.pages_per_seq;
  // Its columns' pages first, then their means, then the sums.
  constexpr int kEach = kColumns * 16 / kThreads;
  const int* const table = c.table + (long)token.b * c.pages_per_seq;
  int page[kEach];
  f32x4 m[kEach][E / 4];
#pragma unroll
  for (int i = 0; i < kEach; ++i) page[i] = table[min(c0 + way + 16 * i, tb.hi - 1)];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const bool bad = (unsigned)page[i] >= (unsigned)c.pages;
    const float* from = p.means + ((long)(bad ? 0 : page[i]) * c.kv_heads + hk) * D + lane * 4;
#pragma unroll
    for (int j = 0; j < E / 4; ++j) m[i][j] = *reinterpret_cast<const f32x4*>(from + 64 * j);
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    double sum = 0.;
#pragma unroll
    for (int j = 0; j < E / 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum = fma(q[4 * j + e], (double)m[i][j][e], sum);
    sum = row16_sum(sum);
    const int col = c0 + way + 16 * i;
    if (lane == 0 && col >= tb.lo && col < tb.hi) scores[col] = (unsigned)page[i] < (unsigned)c.pages ? sortable(sum) : 0;
  }
}

// Tiles of 16 tokens of a sequence, for many of them: a sequence's tiles start at offset / 16 + index.
struct TokenTile {
  int b, t0, count;
  long pos;  // of the first one
  template <typename P> __device__ __forceinline__ TokenTile(const P& p, int slot) {
    const CacheShape& c = p.at;
    auto first_slot = [&](int s) { return packed_begin(c, s) / 16 + s; };
    b = last_at_or_before(c.batch, slot, first_slot);
    const int begin = packed_begin(c, b), end = packed_begin(c, b + 1);
    const long at = begin + 16l * (slot - first_slot(b));  // (a wrong slot's too)
    t0 = (int)at;
    count = at < begin || at >= end ? 0 : (int)(end - at < 16 ? end - at : 16);
    pos = (long)max(0, c.lengths[b]) - (end - at);
  }
};

// Scores of a tile's tokens against columns [c0, c1) by matrix products of 64 bits, 16 columns a wave at a time:
// put(row, column, key). Lane (n, g) holds columns g D / 4 on of q's row n and of a page's mean, of which the
// products take one each in turn; it gets rows g + 4 i of column n.
typedef double f64x4 __attribute__((ext_vector_type(4)));
template <typename T, int D, typename F>
__device__ __forceinline__ void score_tile(const BlockSelectParams<T>& p, const TokenTile& tile, int hk, int c0, int c1, F&& put) {
  constexpr int K = D / 4;
  const CacheShape& c = p.at;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, group = p.heads / c.kv_heads;
  double q[K] = {};
  const T* row = p.q + ((long)(tile.t0 + min(n, tile.count - 1)) * p.heads + hk * group) * D + g * K;
  for (int h = 0; h < group; ++h, row += D)
#pragma unroll
    for (int k = 0; k < K; k += 8) {
      const V8<T> x = *reinterpret_cast<const V8<T>*>(row + k);
#pragma unroll
      for (int e = 0; e < 8; ++e) q[k + e] += (double)(float)x[e];
    }
  // A step's means are loaded a step ahead, their pages another one.
  constexpr int kStep = 16 * (kThreads / 64);
  const int* const table = c.table + (long)tile.b * c.pages_per_seq;
  auto page_of = [&](int col0) { return table[min(col0 + n, c1 - 1)]; };
  f32x4 m[K / 4];
  auto load = [&](int page) {
    const float* from = p.means + ((long)((unsigned)page < (unsigned)c.pages ? page : 0) * c.kv_heads + hk) * D + g * K;
#pragma unroll
    for (int k = 0; k < K / 4; ++k) m[k] = *reinterpret_cast<const f32x4*>(from + 4 * k);
  };
  int col0 = c0 + 16 * (int)(threadIdx.x >> 6);
  if (col0 >= c1) return;
  int page = page_of(col0), ahead = page_of(col0 + kStep);
  load(page);
  for (; col0 < c1; col0 += kStep) {
    f64x4 sum = {0., 0., 0., 0.};
    f32x4 x[K / 4];
#pragma unroll
    for (int k = 0; k < K / 4; ++k) x[k] = m[k];
    const bool bad = (unsigned)page >= (unsigned)c.pages;
    page = ahead;
    ahead = page_of(col0 + 2 * kStep);
    if (col0 + kStep < c1) load(page);
#pragma unroll
    for (int k = 0; k < K; ++k) sum = __builtin_amdgcn_mfma_f64_16x16x4f64(q[k], (double)x[k / 4][k % 4], sum, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col0 + n < c1) put(g + 4 * i, col0 + n, bad ? 0ul : sortable(sum[i]));
  }
}

// Scores and choice of a tile's tokens in one, with the scores in LDS, of up to COLUMNS columns chosen from.
template <typename T, int D, int COLUMNS> __global__ void __launch_bounds__(kThreads) block_select_tile_kernel(BlockSelectParams<T> p) {
  __shared__ unsigned long s_key[16][COLUMNS + 2];  // (rows apart, so that a column's keys are in different banks)
  const CacheShape& c = p.at;
  const int hk = blockIdx.x % c.kv_heads, slot = blockIdx.x / c.kv_heads;
  const TokenTile tile(p, slot);
  // The lists of packed rows that no sequence has: a slot looks after sixteen rows (there are slots enough).
  const int first = packed_begin(c, 0), behind = packed_begin(c, c.batch);
  for (int i = threadIdx.x; i < 16 * p.blocks; i += kThreads) {
    const long t = 16l * slot + i / p.blocks;
    if (t < c.total && (t < first || t >= behind)) p.chosen[(t * c.kv_heads + hk) * p.blocks + i % p.blocks] = -1;
  }
  if (tile.count <= 0) return;
  const TokenBlocks last(p, tile.pos + tile.count - 1, true);
  const int lo = min(p.first, c.pages_per_seq);
  if (last.by_score()) score_tile<T, D>(p, tile, hk, lo, last.hi, [&](int row, int col, unsigned long key) { s_key[row][col - lo] = key; });
  __syncthreads();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int r = wave; r < tile.count; r += kThreads / 64) {
    const TokenBlocks tb(p, tile.pos + r);
    int* const out = p.chosen + ((long)(tile.t0 + r) * c.kv_heads + hk) * p.blocks;
    write_forced(tb, out, p.blocks, threadIdx.x & 63, 64);
    if (tb.by_score() && tb.room > 0)
      choose_in_wave<COLUMNS / 64>(tb.hi - tb.lo, tb.lo, tb.room, out + tb.lo, [&](int i) { return s_key[r][i]; });
  }
}

// Scores of a tile's tokens, in the slab, into memory, for wider tables: kWide columns a workgroup.
constexpr int kWide = 1024;
template <typename T, int D> __global__ void __launch_bounds__(kThreads) block_score_tile_kernel(BlockSelectParams<T> p) {
  const CacheShape& c = p.at;
  const int hk = blockIdx.x % c.kv_heads;
  const TokenTile tile(p, blockIdx.x / c.kv_heads);
  if (tile.count <= 0 || tile.t0 >= p.token0 + p.tokens || tile.t0 + tile.count <= p.token0) return;
  const TokenBlocks last(p, tile.pos + tile.count - 1, true);
  if (!last.by_score()) return;
  const int c0 = max(last.lo, (int)blockIdx.y * kWide), c1 = min(last.hi, ((int)blockIdx.y + 1) * kWide);
  if (c0 >= c1) return;
  score_tile<T, D>(p, tile, hk, c0, c1, [&](int row, int col, unsigned long key) {
    const int t = tile.t0 + row - p.token0;
    if (row < tile.count && t >= 0 && t < p.tokens) p.scores[((long)t * c.kv_heads + hk) * c.pages_per_seq + col] = key;
  });
}

// A token and key/value head by itself: scores of up to COLUMNS columns in LDS, sixteen lanes a column, of which a wave
// chooses. (32 of 500 columns, H16/4 D64 7.3 us, and 64 of up to 1024, 16 tokens of H32/8 D128 16.2: 5.2 and 12.4 of it the
// scores. Scores in memory and a launch of its own for the choice: 4.3 + 5.2 and 11.5 + 7.0.)
constexpr int kTokenThreads = 1024;
template <typename T, int D, int COLUMNS> __global__ void __launch_bounds__(kTokenThreads) block_select_token_kernel(BlockSelectParams<T> p) {
  constexpr int E = D / 16, kWays = kTokenThreads / 16, kEach = 4;
  __shared__ unsigned long s_key[COLUMNS];
  __shared__ __attribute__((aligned(16))) double s_q[D];
  const CacheShape& c = p.at;
  const int hk = blockIdx.x % c.kv_heads, t = p.token0 + blockIdx.x / c.kv_heads;
  const TokenAt token(c, t);
  const TokenBlocks tb(p, token.pos);
  int* const out = p.chosen + ((long)t * c.kv_heads + hk) * p.blocks;
  write_forced(tb, out, p.blocks, threadIdx.x, kTokenThreads);
  if (!tb.by_score() || tb.room == 0) return;
  const int lane = threadIdx.x % 16, way = threadIdx.x / 16, group = p.heads / c.kv_heads;
  // A step's means are loaded a step ahead, their pages another one.
  const int* const table = c.table + (long)token.b * c.pages_per_seq;
  int page[kEach], ahead[kEach];
  f32x4 m[kEach][E / 4];
  bool bad[kEach];
  auto pages = [&](int c0) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) ahead[i] = table[min(c0 + way + kWays * i, tb.hi - 1)];
  };
  auto load = [&] {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      page[i] = ahead[i];
      bad[i] = (unsigned)page[i] >= (unsigned)c.pages;
      const float* from = p.means + ((long)(bad[i] ? 0 : page[i]) * c.kv_heads + hk) * D + lane * 4;
#pragma unroll
      for (int j = 0; j < E / 4; ++j) m[i][j] = *reinterpret_cast<const f32x4*>(from + 64 * j);
    }
  };
  pages(tb.lo);
  if ((int)threadIdx.x < D) {
    const T* row = p.q + ((long)t * p.heads + hk * group) * D + threadIdx.x;
    double sum = 0.;
#pragma unroll 4
    for (int h = 0; h < group; ++h) sum += (double)(float)row[h * D];
    s_q[threadIdx.x] = sum;
  }
  load();
  __syncthreads();
  double q[E];
#pragma unroll
  for (int j = 0; j < E; ++j) q[j] = s_q[64 * (j / 4) + lane * 4 + j % 4];
  for (int c0 = tb.lo; c0 < tb.hi; c0 += kWays * kEach) {
    double sum[kEach] = {};
    bool none[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      none[i] = bad[i];
#pragma unroll
      for (int j = 0; j < E; ++j) sum[i] = fma(q[j], (double)m[i][j / 4][j % 4], sum[i]);
    }
    if (c0 + kWays * kEach < tb.hi) {
      pages(c0 + kWays * kEach);
      load();
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      sum[i] = row16_sum(sum[i]);
      const int col = c0 + way + kWays * i;
      if (lane == 0 && col < tb.hi) s_key[col - tb.lo] = none[i] ? 0ul : sortable(sum[i]);
    }
  }
  __syncthreads();
  if (threadIdx.x < 64) choose_in_wave<COLUMNS / 64>(tb.hi - tb.lo, tb.lo, tb.room, out + tb.lo, [&](int i) { return s_key[i]; });
}

// ------------------------------------------------------------------ choice from scores in memory

// A wave a token and key/value head, which chooses from up to COLUMNS columns.
template <typename T, int COLUMNS> __global__ void __launch_bounds__(kThreads) block_choose_wave_kernel(BlockSelectParams<T> p) {
  const CacheShape& c = p.at;
  const long i = (long)blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (i >= (long)p.tokens * c.kv_heads) return;
  const int hk = (int)(i % c.kv_heads), t = p.token0 + (int)(i / c.kv_heads);
  const TokenBlocks tb(p, TokenAt(c, t).pos);
  int* const out = p.chosen + ((long)t * c.kv_heads + hk) * p.blocks;
  write_forced(tb, out, p.blocks, threadIdx.x & 63, 64);
  if (!tb.by_score() || tb.room == 0) return;
  const unsigned long* const scores = p.scores + i * c.pages_per_seq + tb.lo;
  choose_in_wave<COLUMNS / 64>(tb.hi - tb.lo, tb.lo, tb.room, out + tb.lo, [&](int j) { return scores[j]; });
}

// A workgroup a token and key/value head, of any number of columns: eight bits of the keys at a time, with a
// histogram.
template <typename T> __global__ void __launch_bounds__(kThreads) block_choose_kernel(BlockSelectParams<T> p) {
  __shared__ int hist[256], box[4], found[3];
  const CacheShape& c = p.at;
  const int hk = blockIdx.x % c.kv_heads, t = p.token0 + blockIdx.x / c.kv_heads;
  const TokenBlocks tb(p, TokenAt(c, t).pos);
  int* const out = p.chosen + ((long)t * c.kv_heads + hk) * p.blocks;
  write_forced(tb, out, p.blocks, threadIdx.x, kThreads);
  if (!tb.by_score() || tb.room == 0) return;
  const unsigned long* const scores = p.scores + (long)blockIdx.x * c.pages_per_seq;
  unsigned long prefix = 0, mask = 0;
  int left = tb.room;
  for (int shift = 56; shift >= 0; shift -= 8) {
    hist[threadIdx.x] = 0;
    __syncthreads();
    for (int col = tb.lo + (int)threadIdx.x; col < tb.hi; col += kThreads) {
      const unsigned long key = scores[col];
      if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1);
    }
    __syncthreads();
    const int bin = 255 - (int)threadIdx.x, mine = hist[bin];
    int total;
    const int before = group_scan<kThreads>(mine, total, box);
    if (before < left && before + mine >= left) {
      found[0] = bin;
      found[1] = before;
      found[2] = mine;
    }
    __syncthreads();
    prefix |= (unsigned long)found[0] << shift;
    mask |= 255ul << shift;
    left -= found[1];
    const bool all = found[2] == left;
    __syncthreads();
    if (all) break;
  }
  // Above the prefix all, of those that have it the first `left`.
  int at = tb.lo;
  for (int col0 = tb.lo; col0 < tb.hi; col0 += kThreads) {
    const int col = col0 + (int)threadIdx.x;
    const unsigned long key = col < tb.hi ? scores[col] & mask : 0;
    const bool equal = col < tb.hi && key == prefix, above = col < tb.hi && key > prefix;
    int equals, takes;
    const int rank = group_scan<kThreads>(equal, equals, box);
    const bool take = above || (equal && rank < left);
    const int place = group_scan<kThreads>(take, takes, box);
    if (take) out[at + place] = col;
    at += takes;
    left = max(0, left - equals);
  }
}

}  // namespace

template <typename C, int D> hipError_t launch_key_means(const KeyMeansParams<C>& p, int workgroups, hipStream_t stream) {
  hipLaunchKernelGGL((key_means_kernel<C, D>), dim3(workgroups), dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

template <typename T, int D> hipError_t launch_block_select(const BlockSelectParams<T>& p_, SelectPlan plan, hipStream_t stream) {
  BlockSelectParams<T> p = p_;
  const int width = p.at.pages_per_seq, most = width - p.first - p.last;  // columns chosen from
  if (plan.tiles && plan.slab == 0) {
    const dim3 grid((unsigned)((long)plan.slots * p.at.kv_heads));
    if (most <= 128)
      hipLaunchKernelGGL((block_select_tile_kernel<T, D, 128>), grid, dim3(kThreads), 0, stream, p);
    else if (most <= 256)
      hipLaunchKernelGGL((block_select_tile_kernel<T, D, 256>), grid, dim3(kThreads), 0, stream, p);
    else if (most <= 512)
      hipLaunchKernelGGL((block_select_tile_kernel<T, D, 512>), grid, dim3(kThreads), 0, stream, p);
    else
      hipLaunchKernelGGL((block_select_tile_kernel<T, D, kFusedColumns>), grid, dim3(kThreads), 0, stream, p);
    return hipGetLastError();
  }
  if constexpr (D <= 128) {  // (select_plan)
    if (plan.slab == 0) {
      const dim3 grid((unsigned)p.at.total * p.at.kv_heads);
      p.token0 = 0;
      if (most <= 256)
        hipLaunchKernelGGL((block_select_token_kernel<T, D, 256>), grid, dim3(kTokenThreads), 0, stream, p);
      else if (most <= 512)
        hipLaunchKernelGGL((block_select_token_kernel<T, D, 512>), grid, dim3(kTokenThreads), 0, stream, p);
      else
        hipLaunchKernelGGL((block_select_token_kernel<T, D, kFusedColumns>), grid, dim3(kTokenThreads), 0, stream, p);
      return hipGetLastError();
    }
  }
  for (p.token0 = 0; p.token0 < p.at.total; p.token0 += plan.slab) {
    p.tokens = p.at.total - p.token0 < plan.slab ? p.at.total - p.token0 : plan.slab;
    const unsigned rows = (unsigned)p.tokens * p.at.kv_heads;
    if (plan.tiles)
      hipLaunchKernelGGL((block_score_tile_kernel<T, D>), dim3((unsigned)((long)plan.slots * p.at.kv_heads), (width + kWide - 1) / kWide),
                         dim3(kThreads), 0, stream, p);
    else
      hipLaunchKernelGGL((block_score_kernel<T, D>), dim3(rows, (width + kColumns - 1) / kColumns), dim3(kThreads), 0, stream, p);
    if (most <= 256)
      hipLaunchKernelGGL((block_choose_wave_kernel<T, 256>), dim3((rows + 3) / 4), dim3(kThreads), 0, stream, p);
    else if (most <= kFusedColumns)
      hipLaunchKernelGGL((block_choose_wave_kernel<T, kFusedColumns>), dim3((rows + 3) / 4), dim3(kThreads), 0, stream, p);
    else
      hipLaunchKernelGGL((block_choose_kernel<T>), dim3(rows), dim3(kThreads), 0, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

#define FHOG_INST(D)                                                                                  \
  template hipError_t launch_key_means<__bf16, D>(const KeyMeansParams<__bf16>&, int, hipStream_t);     \
  template hipError_t launch_key_means<_Float16, D>(const KeyMeansParams<_Float16>&, int, hipStream_t); \
  template hipError_t launch_key_means<e4m3, D>(const KeyMeansParams<e4m3>&, int, hipStream_t);         \
  template hipError_t launch_block_select<__bf16, D>(const BlockSelectParams<__bf16>&, SelectPlan, hipStream_t); \
  template hipError_t launch_block_select<_Float16, D>(const BlockSelectParams<_Float16>&, SelectPlan, hipStream_t);
FHOG_INST(64)
FHOG_INST(128)
FHOG_INST(256)
#undef FHOG_INST

}  // namespace fhog
