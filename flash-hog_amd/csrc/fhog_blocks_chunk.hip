// Attention of many new tokens over chosen blocks of a paged cache (fhog_blocks.h), a block at a time.
//
// A token by itself reads all of its blocks through L2, blocks x page_size keys and values for the few rows of its
// group. Here the lists are turned round: for each sequence, key/value head and column the tokens that chose
// it (as bits), whose rows then fill whole matrix tiles against that one page, read once for 128 of them. Each
// row leaves an unnormalised fp32 output with its maximum and sum for each of its blocks, in the place that its
// list gives it, and a last kernel joins a row's outputs in the order of its list: no atomics on numbers, the
// same bits at every call. Scores, statistics and outputs are fp32; a probability enters the second product in T, half a
// step of rounding a term, as in block_token_kernel.
//
// What bounds it: those outputs, written and read once, 8 (head_dim + 2) bytes for each row and block. 2035 tokens in 4
// sequences, H32/8 D128 bf16, 16 blocks of 64, 540 MB of outputs, us: masks 5, items 6, entries 6, tiles 133, sum 108 (5.0 TB/s).
// 4096 tokens, H12/12 D64 e4m3, 16 blocks, 207 MB: 5, 7, 9, 60, 51. (250 MB at D = 128: tiles 91, without their stores 57.
// A token at a time 583 and 744 in all.)
//
//   block_masks_kernel   64 tokens and a key/value head: which of them chose each column
//   block_items_kernel   tokens of each sequence, head and column: how many, in tiles of 128 rows
//   block_entries_kernel who they are, in order
//   block_tile_kernel    a tile: rows of q, scores, probabilities, outputs
//   block_sum_kernel     the join
#include "fhog_blocks.h"

namespace fhog {

namespace {

constexpr float kBound = 256.f;  // bound on an unnormalised probability
constexpr int kThreads = 256;

// A packed token's sequence and position; whether it is a sequence's, and its length within the table.
struct PackedToken {
  int b, pos;
  bool there, beyond;
  template <typename P> __device__ __forceinline__ PackedToken(const P& p, int t) {
    const CacheShape& c = p.at;
    b = last_at_or_before(c.batch, t, [&](int s) { return packed_begin(c, s); });
    const int begin = packed_begin(c, b), end = packed_begin(c, b + 1);
    there = t >= begin && t < end;
    const int length = max(0, c.lengths[b]);
    beyond = length > (long)c.pages_per_seq << c.page_shift;
    pos = length - (end - t);
  }
  // Whether a column shows the token anything.
  __device__ __forceinline__ bool sees(const CacheShape& c, int col) const {
    return there && col >= 0 && col < c.pages_per_seq && (long)col << c.page_shift <= pos;
  }
};

// Tokens of sequence b among the slab's.
template <typename P> __device__ __forceinline__ IndexRange tokens_of(const P& p, int b) {
  return slab_range(packed_begin(p.at, b), packed_begin(p.at, b + 1), p.token0, p.tokens);
}
// The bits of group `group` that are tokens [begin, end).
__device__ __forceinline__ unsigned long group_bits(int group, int begin, int end) {
  const int lo = max(begin - 64 * group, 0), hi = min(end - 64 * group, 64);
  if (lo >= hi) return 0;
  const unsigned long below = hi >= 64 ? ~0ul : (1ul << hi) - 1;
  return below & ~((1ul << lo) - 1);
}

// (256 / 512 / 1024 threads, us in all three, 2035 tokens of 8 heads 20 / 17 / 17, 4096 of 12 24 / 21 / 24)
constexpr int kListThreads = 512;
template <typename T, typename C> __global__ void __launch_bounds__(kListThreads) block_masks_kernel(BlockChunkParams<T, C> p) {
  extern __shared__ unsigned long s_mask[];  // (columns)
  __shared__ PackedTokenAt s_token[64];
  __shared__ unsigned long s_falling;
  const CacheShape& c = p.at;
  const int group = blockIdx.x, hk = blockIdx.y, width = c.pages_per_seq;
  const int count = min(64, p.tokens - 64 * group);
  // Lists and their tokens agree on whose a token is only if the offsets rise. If they do not, nothing is listed,
  // and the rows become NaN (block_sum_kernel).
  bool falls = false;
  for (int i = threadIdx.x; i < c.batch; i += kListThreads) falls = falls || packed_begin(c, i + 1) < packed_begin(c, i);
  falls = __syncthreads_or(falls);
  if (group == 0 && hk == 0 && threadIdx.x == 0) {
    p.total[0] = 0;
    p.total[1] = falls;
  }
  if (threadIdx.x == 0) s_falling = 0;
  for (int i = threadIdx.x; i < width; i += kListThreads) s_mask[i] = 0;
  if ((int)threadIdx.x < count) {
    const PackedToken t(p, p.token0 + 64 * group + threadIdx.x);
    s_token[threadIdx.x] = {t.there && !falls ? t.pos : -1};
  }
  __syncthreads();
  for (int i = threadIdx.x; i < count * p.blocks; i += kListThreads) {
    const int t = i / p.blocks, at = i - t * p.blocks;
    const int* const list = p.chosen + ((long)(p.token0 + 64 * group + t) * c.kv_heads + hk) * p.blocks;
    const int col = list[at];
    if (col < 0 || col >= width || (long)col << c.page_shift > s_token[t].pos) continue;
    atomicOr(&s_mask[col], 1ul << t);
    if (at > 0 && (list[at - 1] < 0 || list[at - 1] >= col)) atomicOr(&s_falling, 1ul << t);
  }
  __syncthreads();
  unsigned long* const out = p.masks + ((long)hk * p.groups + group) * width;
  for (int i = threadIdx.x; i < width; i += kListThreads) out[i] = s_mask[i];
  if (threadIdx.x == 0) p.falling[(long)hk * p.groups + group] = s_falling;
}

// Eight threads a list, each an eighth of the groups, and then the first: the list's tiles get places behind
// others', a wave at a time (in any order: each tile's outputs have places of their own).
template <typename T, typename C> __global__ void __launch_bounds__(kListThreads) block_items_kernel(BlockChunkParams<T, C> p) {
  constexpr int kWays = kListThreads / 64;
  __shared__ int s_count[kWays][64];
  const CacheShape& c = p.at;
  const int way = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int i = blockIdx.x * 64 + lane, width = c.pages_per_seq, group = p.heads / c.kv_heads;
  int count = 0, col = 0, hk = 0, b = 0;
  IndexRange of{0, 0}, groups{0, 0};
  long at = 0;
  if (i < p.lists) {
    col = i % width, hk = i / width % c.kv_heads, b = i / width / c.kv_heads;
    of = tokens_of(p, b);
    groups = list_groups(of, way, kWays);
    at = (long)hk * p.groups * width + col;
  }
#pragma unroll 8
  for (int g = groups.begin; g < groups.end; ++g) count += __popcll(p.masks[at + (long)g * width] & group_bits(g, of.begin, of.end));
  s_count[way][lane] = count;
  __syncthreads();
  int earlier = 0;
  for (int w = 0; w < way; ++w) earlier += s_count[w][lane];
  // (a group that begins with an earlier sequence's tokens is that one's: this one's count there is 0)
#pragma unroll 8
  for (int g = groups.begin; g < groups.end; ++g) {
    if (g > of.begin / 64) p.before[at + (long)g * width] = earlier;
    earlier += __popcll(p.masks[at + (long)g * width] & group_bits(g, of.begin, of.end));
  }
  if (way > 0) return;
  count = 0;
  for (int w = 0; w < kWays; ++w) count += s_count[w][lane];
  const int each = tile_tokens(group), tiles = (count + each - 1) / each;
  int sum, first = 0;
  const int before = wave_scan(tiles, sum);
  if (lane == 0) first = atomicAdd(p.total, sum);
  first = __shfl(first, 0, 64) + before;
  if (count == 0) return;
  p.base[i] = first;
  BlockItem item{};
  item.page = c.table[(long)b * width + col];
  item.hk = hk;
  item.key0 = col << c.page_shift;
  // (a token's position is its index in the packed rows, less its sequence's end, plus the length)
  item.shift = max(0, c.lengths[b]) - packed_begin(c, b + 1) + p.token0;
  for (int k = 0; k < tiles; ++k) {
    item.rows = min(each, count - k * each) * group;
    p.items[first + k] = item;
  }
}

// A thread an element of the tokens' lists, at its rank among the tokens that chose the same.
template <typename T, typename C> __global__ void __launch_bounds__(kListThreads) block_entries_kernel(BlockChunkParams<T, C> p) {
  __shared__ PackedTokenAt s_token[64];
  __shared__ int s_b[64];
  __shared__ IndexRange s_of[64];
  const CacheShape& c = p.at;
  const int group = blockIdx.x, hk = blockIdx.y, width = c.pages_per_seq;
  const int count = min(64, p.tokens - 64 * group);
  if ((int)threadIdx.x < count) {
    const PackedToken t(p, p.token0 + 64 * group + threadIdx.x);
    s_token[threadIdx.x] = {t.there ? t.pos : -1};
    s_b[threadIdx.x] = t.b;
    s_of[threadIdx.x] = tokens_of(p, t.b);
  }
  const unsigned long falling = p.falling[(long)hk * p.groups + group];
  const int each = tile_tokens(p.heads / c.kv_heads);
  __syncthreads();
  for (int i = threadIdx.x; i < count * p.blocks; i += kListThreads) {
    const int t = i / p.blocks, at = i - t * p.blocks;
    const int* const list = p.chosen + ((long)(p.token0 + 64 * group + t) * c.kv_heads + hk) * p.blocks;
    const int col = list[at];
    if (col < 0 || col >= width || (long)col << c.page_shift > s_token[t].pos) continue;
    if (falling >> t & 1) {
      int first = 0;
      while (list[first] != col) ++first;
      if (first < at) continue;
    }
    const int begin = s_of[t].begin, end = s_of[t].end;
    const long place = ((long)hk * p.groups + group) * width + col;
    const unsigned long mask = p.masks[place], bits = mask & group_bits(group, begin, end) & ((1ul << t) - 1);
    if (!(mask >> t & 1)) continue;  // (nothing is listed)
    const int before = group > begin / 64 ? p.before[place] : 0;
    const int rank = before + (int)__popcll(bits), tile = p.base[((long)s_b[t] * c.kv_heads + hk) * width + col] + rank / each;
    p.entries[(long)tile * kTileRows + rank % each] = {64 * group + t, at};
  }
}

// Up to 128 rows of tokens that chose one column, 32 a wave; row r of a tile is its token r / group, head r % group.
// kPast: the outputs are stored past the caches (kCacheBytes; in a branch of one kernel the stores would become one).
template <typename T, typename C, int D, bool kPast>
__global__ void __launch_bounds__(kThreads)
__attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : D == 128 ? 3 : 4)))
block_tile_kernel(BlockChunkParams<T, C> p) {
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int kSwz = D == 64 ? kSwzPairs : kSwzWide;
  typedef PageTile<T, C, D, kThreads, kSwz> Tile;
  constexpr int kStage = 2 * Tile::kTileBytes;
  constexpr int kTurn = 32 * 36;  // floats of a wave's 32 x 32 outputs, rows apart by 36 (16 bytes more than 32)
  constexpr int kLds = 2 * kStage > 4 * kTurn * 4 ? 2 * kStage : 4 * kTurn * 4;
  __shared__ __attribute__((aligned(1024))) char s_kv[kLds];
  __shared__ BlockEntryAt s_entry[kTileRows];

  const CacheShape& c = p.at;
  const int group = p.heads / c.kv_heads, page_rows = 1 << c.page_shift;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 31, g = lane >> 5;
  const bool negate = p.scale < 0.f;  // applied as |scale| to -q (negation is exact)
  const float c2 = fabsf(p.scale) * kLog2e;
  std::conditional_t<D == 64, SwzFrags<T, D>, WideFrags<T, D>> fr;
  fr.init(lane);
  const uint32_t lds = lds_base_u32(s_kv);

  // An eighth of the tiles, which are ordered by sequence and head, to each XCD: its L2 has their queries, and the keys of
  // tiles of one list. (94 us before, 62 at D = 64; runs of 16 / 64 / 256 tiles a XCD 92 / 95 / 107. A workgroup that took
  // tile after tile, the next one's description a tile ahead, took 92 where this took 94, and 79 for 63.)
  const int all = p.total[0], each = (all + 7) / 8, index = blockIdx.x % 8 * each + blockIdx.x / 8;
  if ((int)blockIdx.x / 8 >= each || index >= all) return;
  const BlockItem item = p.items[index];
  const BlockEntryAt entry = p.entries[(long)index * kTileRows + threadIdx.x % kTileRows];
  const int hk = item.hk, rows = item.rows, count = rows / group;  // tokens
  if ((int)threadIdx.x < count) s_entry[threadIdx.x] = entry;
  const bool bad = (unsigned)item.page >= (unsigned)c.pages;
  const long line0 = ((long)(bad ? 0 : item.page) * c.kv_heads + hk) << c.page_shift;
  auto seen_by = [&](int token) { return (int)min((long)token + item.shift + 1 - item.key0, (long)page_rows); };
  __syncthreads();
  const int most = __builtin_amdgcn_readfirstlane(seen_by(s_entry[count - 1].token));  // (tokens rise)

  const bool any = 32 * wave < rows;
  const int row = min(32 * wave + n, rows - 1);
  const int token = row / group, head = row - token * group;
  const int seen = seen_by(s_entry[token].token);
  // Tiles of 32 keys, two stages: a tile is stored while the one before is worked on.
  const int tiles = (most + 31) / 32;
  Tile tile;
  auto fetch = [&](int t) {
    const int left = most - 32 * t;
    // (a page of 16 rows fills the first half only)
    const HalfRows at{{line0 + 32l * t, left > 16 ? line0 + 32l * t + 16 : line0 + 32l * t},
                      {min(15, left - 1), left > 16 ? min(15, left - 17) : min(15, left - 1)}};
    tile.fetch(p.cache, at, threadIdx.x);
  };
  fetch(0);
  V8<T> qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    qf[ks] = *reinterpret_cast<const V8<T>*>(
        p.q + ((long)(p.token0 + s_entry[token].token) * p.heads + hk * group + head) * D + 16 * ks + 8 * g);
    if (negate) qf[ks] = -qf[ks];
  }

  float m = -1e30f, lpart = 0.f;
  f32x16 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = zero16();

  tile.store(lds, threadIdx.x);
  if (tiles > 1) fetch(1);
  __syncthreads();
  for (int t = 0; t < tiles; ++t) {
    const uint32_t sa = lds + (t & 1) * kStage;
    if (t + 1 < tiles) {
      tile.store(lds + ((t + 1) & 1) * kStage, threadIdx.x);
      if (t + 2 < tiles) fetch(t + 2);
    }
    if (any) {
      f32x16 S = zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) S = mma<T>(fr.rowf(sa, 0, ks), qf[ks], S);
      const int left = seen - 32 * t;
      if (__any(left < 32)) {
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (crow(j, g) >= left) S[j] = -INFINITY;
      }
      f32x16 P;
      auto probabilities = [&] {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          P[j] = exp2_fast(fmaf(S[j], c2, -m));  // masked: exp2(-inf) = 0
          sum += P[j];
        }
        return sum;
      };
      float psum = probabilities();
      if (__any(!(psum <= kBound))) {
        float top = S[0];
#pragma unroll
        for (int j = 1; j < 16; ++j) top = fmaxf(top, S[j]);
        const float mnew = fmaxf(m, xgroup_max(top * c2));
        const float alpha = exp2_fast(m - mnew);
        lpart *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
        m = mnew;
        psum = probabilities();
      }
      lpart += psum;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const V8<T> oP = cvt8<T>(s ? hi8(P) : lo8(P));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] = mma<T>(fr.trf(sa, Tile::kTileBytes, dt, s), oP, acc[dt]);
      }
    }
    __syncthreads();
  }
  if (!any) return;
  if (bad) lpart = NAN;
  const float l = xgroup_sum(lpart);
  // Each row to its place, 128 bytes of it at a time: 32 x 32 outputs turned in LDS, in place of the tiles (all
  // waves are behind the last barrier, and each has a part of its own).
  const int mine = min(32, rows - 32 * wave);
  auto place = [&](int r) {  // of row r of this wave: the index of its outputs
    const int at = 32 * wave + r, tk = at / group;
    return ((long)(s_entry[tk].token * c.kv_heads + hk) * p.blocks + s_entry[tk].slot) * group + at - tk * group;
  };
  if (lane < mine) {
    // (rows n of both lane groups have the same m and l)
    float* ml = p.parts_ml + 2 * place(lane);
    ml[0] = m;
    ml[1] = l;
  }
  float* const turn = reinterpret_cast<float*>(s_kv) + wave * kTurn;
  long to[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) to[i] = place(min(8 * i + (lane >> 3), mine - 1)) * D + 4 * (lane & 7);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    __builtin_amdgcn_wave_barrier();  // (a wave's LDS operations run in order; only the compiler could move them)
#pragma unroll
    for (int a = 0; a < 4; ++a)
      *reinterpret_cast<f32x4*>(turn + n * 36 + 8 * a + 4 * g) =
          f32x4{acc[dt][4 * a], acc[dt][4 * a + 1], acc[dt][4 * a + 2], acc[dt][4 * a + 3]};
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (8 * i + (lane >> 3) < mine) {
        f32x4* const at = reinterpret_cast<f32x4*>(p.parts + to[i] + 32 * dt);
        const f32x4 x = *reinterpret_cast<const f32x4*>(turn + (8 * i + (lane >> 3)) * 36 + 4 * (lane & 7));
        if constexpr (kPast)
          __builtin_nontemporal_store(x, at);
        else
          *at = x;
      }
  }
}

// Joins the rows' blocks, each row's in the order of its list: four columns a thread, whole rows. A wave forms the
// weights 2^(m - top) / sum of every fourth row first, in LDS. A column that a list names twice has the outputs
// of its first place there.
template <typename T, typename C, int D> __global__ void __launch_bounds__(kThreads) block_sum_kernel(BlockChunkParams<T, C> p) {
  constexpr int kLanes = D / 4, R = kThreads / kLanes;
  __shared__ int s_from[R][kSumBlocks];
  __shared__ float s_w[R][kSumBlocks];
  __shared__ int s_count[R];
  const CacheShape& c = p.at;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = p.heads / c.kv_heads;
  const long rows = (long)p.tokens * p.heads, row0 = (long)blockIdx.x * R;
  // A row's first place among the outputs; its others are `group` apart.
  auto place = [&](long row) {
    const long token = row / p.heads;
    const int h = (int)(row - token * p.heads), hk = h / group;
    return (token * c.kv_heads + hk) * p.blocks * group + h - hk * group;
  };
  for (int r = wave; r < R && row0 + r < rows; r += 4) {
    const long row = row0 + r;
    const int token = (int)(row / p.heads), hk = (int)(row - (long)token * p.heads) / group;
    const PackedToken pt(p, p.token0 + token);
    const int* const list = p.chosen + ((long)(p.token0 + token) * c.kv_heads + hk) * p.blocks;
    const float* const ml = p.parts_ml + 2 * place(row);
    int count = 0;
    float top = -INFINITY, sum = 0.f;
    bool rises = true;
    for (int i0 = 0; i0 < p.blocks; i0 += 64) {
      const int i = i0 + lane, col = i < p.blocks ? list[i] : -1;
      const bool sees = pt.sees(c, col);
      int from = i;
      const int before = i > 0 && i < p.blocks ? list[i - 1] : 0;
      rises = rises && !__any(sees && i > 0 && (before < 0 || before >= col));
      if (!rises) {
        from = 0;
        while (sees && list[from] != col) ++from;
      }
      const unsigned long all = __ballot(sees);
      if (sees) {
        const int at = count + __popcll(all & ((1ul << lane) - 1));
        s_from[r][at] = from;
        const float m = ml[2l * from * group];
        s_w[r][at] = m;
        top = fmaxf(top, m);
      }
      count += __popcll(all);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    for (int i = lane; i < count; i += 64) {
      const float w = exp2_fast(s_w[r][i] - top);
      sum += w * ml[2l * s_from[r][i] * group + 1];
      s_w[r][i] = w;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    for (int i = lane; i < count; i += 64) s_w[r][i] *= inv;
    // a row that sees nothing: 0; a length beyond the table: NaN; no sequence's: 0, or left as it is; offsets that do
    // not rise: NaN
    if (lane == 0) s_count[r] = p.total[1] ? -1 : pt.there ? (pt.beyond ? -1 : count) : p.clear_rest ? 0 : -2;
  }
  __syncthreads();
  const int r = threadIdx.x / kLanes, column = 4 * (int)(threadIdx.x % kLanes);
  const long row = row0 + r;
  if (row >= rows) return;
  const int count = s_count[r];
  if (count == -2) return;
  f32x4 o = zero4();
  const float* const from = p.parts + place(row) * D + column;
  const long apart = (long)group * D;
#pragma unroll 8
  for (int i = 0; i < count; ++i) o += s_w[r][i] * __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(from + s_from[r][i] * apart));
  if (count == -1) o = f32x4{NAN, NAN, NAN, NAN};
  *reinterpret_cast<V4<T>*>(p.out + ((long)p.token0 * p.heads + row) * D + column) = cvt4<T>(o);
}

}  // namespace

template <typename T, typename C, int D>
hipError_t launch_block_chunk(const BlockChunkParams<T, C>& p_, int slab, hipStream_t stream) {
  BlockChunkParams<T, C> p = p_;
  for (p.token0 = 0; p.token0 < p.at.total; p.token0 += slab) {
    p.tokens = p.at.total - p.token0 < slab ? p.at.total - p.token0 : slab;
    p.groups = (p.tokens + 63) / 64;
    const long most = (long)p.tokens * p.blocks * p.at.kv_heads / tile_tokens(p.heads / p.at.kv_heads) + p.lists;
    hipLaunchKernelGGL((block_masks_kernel<T, C>), dim3(p.groups, p.at.kv_heads), dim3(kListThreads),
                       p.at.pages_per_seq * sizeof(unsigned long), stream, p);
    hipLaunchKernelGGL((block_items_kernel<T, C>), dim3((p.lists + 63) / 64), dim3(kListThreads), 0, stream, p);
    hipLaunchKernelGGL((block_entries_kernel<T, C>), dim3(p.groups, p.at.kv_heads), dim3(kListThreads), 0, stream, p);
    const dim3 tiles((unsigned)((most + 7) / 8 * 8));
    if ((long)p.tokens * p.heads * p.blocks * D * 4 > kCacheBytes)
      hipLaunchKernelGGL((block_tile_kernel<T, C, D, true>), tiles, dim3(kThreads), 0, stream, p);
    else
      hipLaunchKernelGGL((block_tile_kernel<T, C, D, false>), tiles, dim3(kThreads), 0, stream, p);
    constexpr long R = kThreads / (D / 4);
    hipLaunchKernelGGL((block_sum_kernel<T, C, D>), dim3((unsigned)(((long)p.tokens * p.heads + R - 1) / R)), dim3(kThreads), 0,
                       stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

#define FHOG_INST(T, C, D) template hipError_t launch_block_chunk<T, C, D>(const BlockChunkParams<T, C>&, int, hipStream_t);
FHOG_INST(__bf16, __bf16, 64)
FHOG_INST(__bf16, __bf16, 128)
FHOG_INST(__bf16, __bf16, 256)
FHOG_INST(__bf16, e4m3, 64)
FHOG_INST(__bf16, e4m3, 128)
FHOG_INST(__bf16, e4m3, 256)
FHOG_INST(_Float16, _Float16, 64)
FHOG_INST(_Float16, _Float16, 128)
FHOG_INST(_Float16, _Float16, 256)
FHOG_INST(_Float16, e4m3, 64)
FHOG_INST(_Float16, e4m3, 128)
FHOG_INST(_Float16, e4m3, 256)
#undef FHOG_INST

}  // namespace fhog
