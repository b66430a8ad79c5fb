// Attention of new tokens over a paged key/value cache (fhog_paged.h): O = softmax(scale q K^T) V
// for the packed new tokens of several sequences, each against its own sequence's cached
// keys up to its own position, optionally the last `window` of them and the first `sinks`.
//
// Query heads that share a key/value head are taken together: row r of a sequence's tile is
// token r / group, head r % group, so a cached row is read once for the whole group.
// Scores are formed transposed (keys x rows), so that a lane holds one row's scores, and
// the output as O^T = V^T P^T, as in the dense forward; one sweep with the running maximum
// and sum, rescaled only when a row's probabilities exceed 2^8.
//
// paged_token_kernel, for few rows a sequence: 16 rows a workgroup, whose waves take every
// kWaves-th tile of 32 keys each on their own, through LDS of their own (no barrier in
// the sweep), and join at the end.
// paged_chunk_kernel, for many: 32 rows a wave, 128 rows a workgroup, all its waves on the same
// tile, or 64 rows and two tiles at a time. Tiles that see most keys go first: a sequence's last, or
// on grids of a few rounds those of all sequences, sorted by each workgroup for itself. 2-byte rows
// go to LDS by DMA (8 sequences of 17 to 512 new tokens, 32 heads over 8, D = 128, window 2048:
// 138.5 us through registers, 121.8 so).
//
// Scores, maxima, sums and running outputs are fp32. A probability enters the second product in T, because
// the matrix instructions take both operands in it: one rounding of half a step a term, while
// the row's sum is of the unrounded ones. The outputs' 2-norm error is 1.0 to 1.2 times that of fp32
// probabilities rounded once at the end (bf16 1.7e-3 to 1.9e-3); two terms a probability would double
// that product.
//
// Where tiles of rows are few, a sequence's keys are dealt to several workgroups (splits of
// split_tiles tiles), which leave unnormalised fp32 outputs with their maxima and sums;
// paged_join_kernel joins them in order. The number of splits follows from sizes that the
// host knows (no length is read back), so a call can be captured; workgroups of splits
// beyond a sequence's end leave at once.
#include "fhog_paged.h"

namespace fhog {

namespace {

constexpr float kBound = 256.f;  // bound on an unnormalised probability

// A workgroup's rows: `rows` of them from row0 of sequence b on.
struct RowTile {
  int b, row0, rows, group;
  int begin;    // packed row of the sequence's first new token
  int pos0;     // that token's position
  int length;   // cut to the table's capacity
  bool beyond;  // the length is beyond it

  template <int ROWS, typename P> __device__ __forceinline__ static RowTile at(const P& p, int slot) {
    const CacheShape& c = p.at;
    const int group = p.heads / c.kv_heads;
    auto first_slot = [&](int b) { return (int)((long)packed_begin(c, b) * group / ROWS) + b; };
    const int b = c.offsets ? last_at_or_before(c.batch, slot, first_slot) : slot / p_slots<ROWS>(group);
    return of<ROWS>(p, b, c.offsets ? slot - first_slot(b) : slot % p_slots<ROWS>(group));
  }
  // Tile `tile` of sequence b.
  template <int ROWS, typename P> __device__ __forceinline__ static RowTile of(const P& p, int b, int tile) {
    const CacheShape& c = p.at;
    RowTile t;
    t.group = p.heads / c.kv_heads;
    t.b = b;
    t.begin = packed_begin(c, t.b);
    const int count = c.offsets ? max(0, packed_begin(c, t.b + 1) - t.begin) : 1;
    // (long: a wrong slot's tile times ROWS)
    const long left = (long)count * t.group - (long)tile * ROWS;
    t.row0 = tile * ROWS;
    t.rows = tile < 0 || left < 0 ? 0 : (int)(left < ROWS ? left : ROWS);
    const long capacity = (long)c.pages_per_seq << c.page_shift;
    const int length = max(0, c.lengths[t.b]);
    t.beyond = length > capacity;
    t.length = t.beyond ? (int)capacity : length;
    t.pos0 = length - count;
    return t;
  }
  // Tiles of a sequence of one token.
  template <int ROWS> __device__ __forceinline__ static int p_slots(int group) { return (group + ROWS - 1) / ROWS; }

  __device__ __forceinline__ int position(int r) const { return pos0 + (row0 + r) / group; }
  // Element offset of row r's head in q and out.
  __device__ __forceinline__ long offset(int r, int hk, int heads, int d) const {
    const int i = (row0 + r) / group, h = (row0 + r) % group;
    return ((long)(begin + i) * heads + hk * group + h) * d;
  }
};

// Zeroes the packed rows behind the last sequence, and those before the first.
template <int D, typename P> __device__ __forceinline__ void clear_rest(const P& p, int worker, int workers, int threads) {
  if (!p.clear_rest || !p.at.offsets) return;
  const long per_row = (long)p.heads * D / 8;
  const long first = (long)packed_begin(p.at, 0) * per_row;
  const long last = (long)packed_begin(p.at, p.at.batch) * per_row, end = (long)p.at.total * per_row;
  const long i0 = (long)worker * threads + threadIdx.x, step = (long)workers * threads;
  u32x4* out = reinterpret_cast<u32x4*>(p.out);
  for (long i = i0; i < first; i += step) out[i] = u32x4{0, 0, 0, 0};
  for (long i = last + i0; i < end; i += step) out[i] = u32x4{0, 0, 0, 0};
}

// The pages of a tile's two halves, loaded a step before the tile's rows are.
struct Pages {
  int page0 = 0, page1 = 0;
  // `zero` is 0 in a vector register: the same address in every lane, but a vector load,
  // which is waited for in order. A scalar one would be waited for with the step's first LDS
  // read.
  __device__ __forceinline__ void load(const CacheShape& c, const PageSpan& span, int b, int t, int zero) {
    const int k0 = span.key(t), rhi = span.last_row(t);
    // (each half's page from a row that is read)
    const int* row = c.table + (long)b * c.pages_per_seq + zero;
    page0 = row[(k0 + span.first_row(t)) >> c.page_shift];
    page1 = row[(k0 + min(rhi, 16)) >> c.page_shift];
  }
  // Replaces pages that are none by page 0; whether there were any.
  __device__ __forceinline__ bool check(const CacheShape& c) {
    const bool bad = (unsigned)page0 >= (unsigned)c.pages || (unsigned)page1 >= (unsigned)c.pages;
    if (bad) page0 = page1 = 0;
    return bad;
  }
};
__device__ __forceinline__ int vector_zero() {
  int zero = 0;
  asm volatile("" : "+v"(zero));
  return zero;
}

// Where split `split` of a tile of rows leaves its output (ROWS rows of D) and, behind all
// outputs, its rows' maxima and sums.
template <int ROWS, int D, typename P> struct Parts {
  float* out;
  float* ml;
  __device__ __forceinline__ Parts(const P& p, int slot, int hk, int split) {
    const long part = ((long)slot * p.at.kv_heads + hk) * p.splits + split;
    const long count = (long)p.slots * p.at.kv_heads * p.splits;
    out = p.parts + part * ROWS * D;
    ml = p.parts + count * ROWS * D + part * ROWS * 2;
  }
};

// ------------------------------------------------------------------ few rows

constexpr int kTokenRows = 16;

template <typename T, typename C, int D, int kWaves>
__global__ void __launch_bounds__(64 * kWaves)
paged_token_kernel(PagedParams<T, C> p) {
  constexpr int ROWS = kTokenRows;
  constexpr int KS = D / 32, DB = D / 16;
  // e4m3 keys go straight into operands (128.0 -> 125.3 us for 16 sequences of up to 32768 keys,
  // 32 heads over 8, D = 128); 2-byte ones, whose operand loads take half lines, through LDS
  // (215 us against 221).
  typedef KeyPieces<T, C, D> Keys;
  constexpr bool kDirect = Keys::kQuantised;
  typedef PageTile<T, C, D, 64, D == 64 ? kSwzRows : kSwzWide, kDirect ? 1 : 2> Tile;
  constexpr int kWaveLds = (kDirect ? 1 : 2) * Tile::kTileBytes;
  __shared__ __attribute__((aligned(1024))) char s_kv[kWaves * kWaveLds];
  __shared__ float s_ml[kWaves][ROWS][2];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int hk = blockIdx.x % p.at.kv_heads, slot = blockIdx.x / p.at.kv_heads, split = blockIdx.y;
  clear_rest<D>(p, blockIdx.x + gridDim.x * blockIdx.y, gridDim.x * gridDim.y, 64 * kWaves);
  const RowTile rt = RowTile::template at<ROWS>(p, slot);
  if (rt.rows <= 0) return;
  const int first_pos = __builtin_amdgcn_readfirstlane(rt.position(0));
  const int last_pos = __builtin_amdgcn_readfirstlane(rt.position(rt.rows - 1));
  const PageSpan span(first_pos, last_pos, rt.length, p.window, p.sinks);
  const int t0 = split * p.split_tiles, t1 = min(span.tiles, t0 + p.split_tiles);
  if (split > 0 && t0 >= t1) return;

  // This lane's row (n): its queries as the score products' B operand, and its position.
  const int r = min(n, rt.rows - 1);
  const int pos = rt.position(r);
  const bool negate = p.scale < 0.f;  // applied as |scale| to -q (negation is exact)
  V8<T> qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    qf[ks] = *reinterpret_cast<const V8<T>*>(p.q + rt.offset(r, hk, p.heads, D) +
                                             (kDirect ? Keys::column(ks, g) : 32 * ks + 8 * g));
    if (negate) qf[ks] = -qf[ks];
  }
  const float c2 = fabsf(p.scale) * kLog2e;

  std::conditional_t<D == 64, SwzFrags16<T, D>, WideFrags16<T, D>> fr;
  fr.init(lane);
  const uint32_t lds = lds_base_u32(s_kv) + wave * kWaveLds;
  float m = -1e30f, lpart = 0.f;
  f32x4 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) acc[db] = zero4();
  bool bad = rt.beyond;

  Keys keys;
  Tile tile;
  Pages pages;
  const int zero = vector_zero();
  // Fetches tile t, whose pages are there, and loads those of this wave's next one.
  auto fetch = [&](int t) {
    bad |= pages.check(p.at);
    const int k0 = span.key(t), rlo = span.first_row(t), rhi = span.last_row(t);
    if constexpr (kDirect)
      keys.fetch(p.cache, hk, p.at.kv_heads, p.at.page_shift, k0, rlo, rhi, pages.page0, pages.page1, n, g);
    tile.fetch(p.cache, hk, p.at.kv_heads, p.at.page_shift, k0, rlo, rhi, pages.page0, pages.page1, lane);
    if (t + kWaves < t1) pages.load(p.at, span, rt.b, t + kWaves, zero);
  };
  int t = t0 + wave;
  if (t < t1) {
    pages.load(p.at, span, rt.b, t, zero);
    fetch(t);
  }
  for (; t < t1; t += kWaves) {
    const int k0 = span.key(t), rlo = span.first_row(t), rhi = span.last_row(t);
    f32x4 S[2];
    auto scores = [&](auto&& keys_of) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        S[kb] = zero4();
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) S[kb] = mma16<T>(keys_of(kb, ks), qf[ks], S[kb]);
      }
    };
    // (before the next tile takes the registers)
    if constexpr (kDirect) scores([&](int kb, int ks) { return keys.operand(kb, ks); });
    __builtin_amdgcn_wave_barrier();  // (the wave's LDS operations run in order; only the compiler could move them)
    tile.store(lds, lane);
    __builtin_amdgcn_wave_barrier();
    if (t + kWaves < t1) fetch(t + kWaves);
    if constexpr (!kDirect) scores([&](int kb, int ks) { return fr.rowf(lds, 0, kb, ks); });
    if (rlo > 0 || rhi < 31 || k0 + 31 > first_pos || (p.window && k0 <= last_pos - p.window)) {
      const int klim = min(rhi, pos - k0);
      const int klow = p.window ? pos - p.window + 1 - k0 : 0, ksinks = p.sinks - k0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int key = 16 * (e >> 2) + 4 * g + (e & 3);
        if (key > klim || key < rlo || (key < klow && key >= ksinks)) S[e >> 2][e & 3] = -INFINITY;
      }
    }
    f32x8 P;
    auto probabilities = [&] {
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        P[e] = exp2_fast(fmaf(S[e >> 2][e & 3], c2, -m));  // masked: exp2(-inf) = 0
        sum += P[e];
      }
      return sum;
    };
    float psum = probabilities();
    if (__any(!(psum <= kBound))) {
      float top = S[0][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, S[e >> 2][e & 3]);
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float mnew = fmaxf(m, top * c2);
      const float alpha = exp2_fast(m - mnew);
      lpart *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) acc[db] *= alpha;
      m = mnew;
      psum = probabilities();
    }
    lpart += psum;
    const V8<T> oP = cvt8<T>(P);
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = mma16<T>(fr.trf(lds, kDirect ? 0 : Tile::kTileBytes, db), oP, acc[db]);
  }

  // The waves' outputs meet in LDS, in place of the tiles: (wave, column, row), so that the
  // lanes of a column block write 16 rows side by side.
  if (__any(bad)) lpart = NAN;
  const float l = group4_sum(lpart);
  __syncthreads();
  float* so = reinterpret_cast<float*>(s_kv);
  static_assert(kWaves * ROWS * D * (int)sizeof(float) <= kWaves * kWaveLds, "the join reuses the tiles");
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i) so[(wave * D + 16 * db + 4 * g + i) * ROWS + n] = acc[db][i];
  if (g == 0) {
    s_ml[wave][n][0] = m;
    s_ml[wave][n][1] = l;
  }
  __syncthreads();
  Parts<ROWS, D, PagedParams<T, C>> parts(p, slot, hk, split);
  for (int i = threadIdx.x; i < ROWS * (D / 4); i += 64 * kWaves) {
    const int row = i / (D / 4), col = 4 * (i % (D / 4));
    if (row >= rt.rows) break;
    float top = s_ml[0][row][0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, s_ml[w][row][0]);
    float sum = 0.f;
    f32x4 o = zero4();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = exp2_fast(s_ml[w][row][0] - top);
      sum += f * s_ml[w][row][1];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += f * so[(w * D + col + j) * ROWS + row];
    }
    if (p.splits > 1) {
      *reinterpret_cast<f32x4*>(parts.out + row * D + col) = o;
      if (col == 0) {
        parts.ml[2 * row] = top;
        parts.ml[2 * row + 1] = sum;
      }
    } else {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing: 0
      *reinterpret_cast<V4<T>*>(p.out + rt.offset(row, hk, p.heads, D) + col) = cvt4<T>(o * inv);
    }
  }
}

// ------------------------------------------------------------------ many rows

// Waves that share a tile of keys, 32 rows each: RW of four; the 4 / RW groups of them take
// every (4 / RW)-th tile and join at the end.
// (128 rows at D = 128: three waves per SIMD, 168 registers and a few of them spilled outside the
// loop, 156 -> 120 us for those 8 sequences.)
template <typename T, typename C, int D, int RW>
__global__ void __launch_bounds__(256)
__attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : D == 64 || RW == 4 ? 3 : 2)))
paged_chunk_kernel(PagedParams<T, C> p) {
  constexpr int ROWS = 32 * RW, KW = 4 / RW;
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int kSwz = D == 64 ? kSwzPairs : kSwzWide;
  typedef PageTile<T, C, D, 64 * RW, kSwz> Tile;
  constexpr bool kDma = sizeof(C) == sizeof(T);
  constexpr int kStage = 2 * Tile::kTileBytes;
  constexpr int kStages = kDma && KW * 3 * kStage <= (D == 256 ? 160 : 53) * 1024 ? 3 : 2;
  __shared__ __attribute__((aligned(1024))) char s_kv[KW * kStages * kStage];
  __shared__ float s_ml[KW][ROWS][2];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rw = wave % RW, kw = wave / RW;
  const int thread = threadIdx.x % (64 * RW);  // of its group
  const int n = lane & 31, g = lane >> 5;
  // (backwards: a sequence's last rows first)
  const int hk = blockIdx.x % p.at.kv_heads, slot = p.slots - 1 - (int)blockIdx.x / p.at.kv_heads, split = blockIdx.y;
  clear_rest<D>(p, blockIdx.x + gridDim.x * blockIdx.y, gridDim.x * gridDim.y, 256);
  RowTile rt;
  if (p.longest_first) {
    int seq, tile;
    if (!longest_first<ROWS>(p.at, p.heads / p.at.kv_heads, p.slots - 1 - slot, lane, seq, tile)) return;
    rt = RowTile::template of<ROWS>(p, seq, tile);
  } else {
    rt = RowTile::template at<ROWS>(p, slot);
  }
  if (rt.rows <= 0) return;
  const int first_pos = __builtin_amdgcn_readfirstlane(rt.position(0));
  const int last_pos = __builtin_amdgcn_readfirstlane(rt.position(rt.rows - 1));
  const PageSpan span(first_pos, last_pos, rt.length, p.window, p.sinks);
  const int t0 = split * p.split_tiles;
  const int t1 = __builtin_amdgcn_readfirstlane(min(span.tiles, t0 + p.split_tiles));
  if (split > 0 && t0 >= t1) return;

  // This wave's rows, from 32 * rw on, and this lane's.
  const bool any = 32 * rw < rt.rows;
  const int wfirst = __builtin_amdgcn_readfirstlane(rt.position(min(32 * rw, rt.rows - 1)));
  const int wlast = __builtin_amdgcn_readfirstlane(rt.position(min(32 * rw + 31, rt.rows - 1)));
  const int row = 32 * rw + n;
  const int r = min(row, rt.rows - 1);
  const int pos = rt.position(r);
  const bool negate = p.scale < 0.f;
  V8<T> qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    qf[ks] = *reinterpret_cast<const V8<T>*>(p.q + rt.offset(r, hk, p.heads, D) + 16 * ks + 8 * g);
    if (negate) qf[ks] = -qf[ks];
  }
  const float c2 = fabsf(p.scale) * kLog2e;

  std::conditional_t<D == 64, SwzFrags<T, D>, WideFrags<T, D>> fr;
  fr.init(lane);
  const uint32_t lds = lds_base_u32(s_kv) + kw * kStages * kStage;
  float m = -1e30f, lpart = 0.f;
  f32x16 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = zero16();
  bool bad = rt.beyond;

  // Tile t, staged at sa, for this wave's rows.
  auto attend = [&](int t, uint32_t sa) {
    const int k0 = span.key(t);
    // a wave's own positions: nothing before its window's start or behind its last row
    const bool active = any && k0 <= wlast &&
                        (t < span.sink_tiles || !p.window || k0 + 31 > wfirst - p.window || k0 < p.sinks);
    if (active) {
      f32x16 S = zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) S = mma<T>(fr.rowf(sa, 0, ks), qf[ks], S);
      const int rlo = span.first_row(t), rhi = span.last_row(t);
      if (rlo > 0 || rhi < 31 || k0 + 31 > wfirst || (p.window && k0 <= wlast - p.window)) {
        asm volatile("");  // (a branch: the compiler would take the masks' instructions into every tile)
        const int klim = min(rhi, pos - k0);
        const int wlow = p.window && t >= span.sink_tiles ? pos - p.window + 1 - k0 : 0, klow = max(rlo, wlow);
        if (t >= span.sink_tiles && p.sinks - k0 > rlo) {  // sinks among the window's keys
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int key = crow(j, g);
            if (key > klim || key < rlo || (key < klow && key >= p.sinks - k0)) S[j] = -INFINITY;
          }
        } else {
          // klow <= key <= klim as one comparison; no key if there is none between
          const int from = crow(0, g) - (klow <= klim ? klow : 64);
          const unsigned most = (unsigned)max(klim - klow, 0);
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if ((unsigned)(from + crow(j, 0)) > most) S[j] = -INFINITY;
        }
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
  };

  const int steps = (t1 - t0 + KW - 1) / KW;
  const int mine = t0 + kw;
  if constexpr (kDma) {
    // A ring of kStages tiles, filled by LDS DMAs. Where the tiles begin comes through LDS too, for
    // kAhead steps at a time: a load from global memory in the loop would wait for the DMAs.
    constexpr int kAhead = 128 / KW;
    typedef PageDma<T, D, 64 * RW, kSwz> Dma;
    __shared__ typename Dma::Place s_at[KW][kAhead];
    const Dma dma(rw, lane);
    for (int s0 = 0; s0 < steps; s0 += kAhead) {
      const int first = mine + KW * s0, rounds = min(kAhead, steps - s0);
      const int count = min(rounds, (t1 - first + KW - 1) / KW);  // this group's tiles (may be below zero)
      if (s0 > 0) __syncthreads();
      for (int i = thread; i < count; i += 64 * RW) {
        const int t = first + KW * i;
        Pages pages;
        pages.load(p.at, span, rt.b, t, 0);
        s_at[kw][i] = Dma::place(p.at, hk, span.key(t), span.first_row(t), span.last_row(t), pages.page0, pages.page1);
      }
      wait_vmem();
      __syncthreads();
      auto issue = [&](int i, const typename Dma::Place& place) {
        typename Dma::Place at;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)place.half[h]);
          const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(place.half[h] >> 32));
          at.half[h] = (long)((unsigned long)hi << 32 | lo);
        }
        bad |= (at.half[0] & 1) != 0;
        const int t = first + KW * i;
        dma.issue(lds + (uint32_t)(i % kStages) * kStage, p.cache, at, span.first_row(t), span.last_row(t));
      };
#pragma unroll
      for (int i = 0; i < kStages - 1; ++i)
        if (i < count) issue(i, s_at[kw][i]);
      typename Dma::Place next = s_at[kw][min(kStages - 1, kAhead - 1)];  // (a step ahead of its use)
      for (int i = 0; i < rounds; ++i) {
        wait_tile<kStages, Dma::kLoads>(i, count);
        __syncthreads();
        if (i + kStages - 1 < count) issue(i + kStages - 1, next);
        next = s_at[kw][min(i + kStages, kAhead - 1)];
        if (i < count) attend(first + KW * i, lds + (uint32_t)(i % kStages) * kStage);
      }
    }
    __syncthreads();
  } else {
    Tile tile;
    Pages pages;
    const int zero = vector_zero();
    // Fetches tile t, whose pages are there, and loads those of this group's next one.
    auto fetch = [&](int t) {
      bad |= pages.check(p.at);
      tile.fetch(p.cache, hk, p.at.kv_heads, p.at.page_shift, span.key(t), span.first_row(t), span.last_row(t),
                 pages.page0, pages.page1, thread);
      if (t + KW < t1) pages.load(p.at, span, rt.b, t + KW, zero);
    };
    // In step i a group works on tile t0 + kw + KW i, if there is one. It was stored to stage
    // i % 2 in step i - 1, whose barrier at its end shows it; the stage's last readers passed the
    // barrier of step i - 2.
    if (mine < t1) {
      pages.load(p.at, span, rt.b, mine, zero);
      fetch(mine);
      tile.store(lds, thread);
      if (mine + KW < t1) fetch(mine + KW);
    }
    __syncthreads();
    for (int i = 0; i < steps; ++i) {
      const int t = mine + KW * i;
      if (t + KW < t1) {
        tile.store(lds + ((i + 1) & 1) * kStage, thread);
        if (t + 2 * KW < t1) fetch(t + 2 * KW);
      }
      if (t < t1) attend(t, lds + (i & 1) * kStage);
      __syncthreads();
    }
  }

  if (bad) lpart = NAN;
  float l = xgroup_sum(lpart);
  if constexpr (KW > 1) {
    // The other groups hand their sums to the first, in LDS in place of the tiles.
    static_assert((KW - 1) * RW * DT * 4096 <= KW * kStages * kStage, "the join reuses the tiles");
    float* box = reinterpret_cast<float*>(s_kv) + 4 * lane;
    auto place = [&](int k, int dt, int a) { return box + 256 * (((k - 1) * RW + rw) * DT * 4 + 4 * dt + a); };
    if (kw > 0) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int a = 0; a < 4; ++a)
          *reinterpret_cast<f32x4*>(place(kw, dt, a)) =
              f32x4{acc[dt][4 * a], acc[dt][4 * a + 1], acc[dt][4 * a + 2], acc[dt][4 * a + 3]};
      if (g == 0) {
        s_ml[kw][row][0] = m;
        s_ml[kw][row][1] = l;
      }
    }
    __syncthreads();
    if (kw > 0) return;
#pragma unroll
    for (int k = 1; k < KW; ++k) {
      const float mk = s_ml[k][row][0], top = fmaxf(m, mk);
      const float f = exp2_fast(m - top), fk = exp2_fast(mk - top);
      l = l * f + s_ml[k][row][1] * fk;
      m = top;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const f32x4 y = *reinterpret_cast<const f32x4*>(place(k, dt, a));
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[dt][4 * a + j] = acc[dt][4 * a + j] * f + y[j] * fk;
        }
    }
  }
  if (row >= rt.rows) return;
  if (p.splits > 1) {
    Parts<ROWS, D, PagedParams<T, C>> parts(p, slot, hk, split);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int a = 0; a < 4; ++a)
        *reinterpret_cast<f32x4*>(parts.out + row * D + 32 * dt + 8 * a + 4 * g) =
            f32x4{acc[dt][4 * a], acc[dt][4 * a + 1], acc[dt][4 * a + 2], acc[dt][4 * a + 3]};
    if (g == 0) {
      parts.ml[2 * row] = m;
      parts.ml[2 * row + 1] = l;
    }
  } else {
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing: 0
    T* o = p.out + rt.offset(row, hk, p.heads, D);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        f32x4 x;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = acc[dt][4 * a + j] * inv;
        *reinterpret_cast<V4<T>*>(o + 32 * dt + 8 * a + 4 * g) = cvt4<T>(x);
      }
  }
}

// ------------------------------------------------------------------ the splits' join

// One workgroup a tile of rows and key/value head. Its rows' weights 2^(m - top) / sum come
// first, in LDS; then each thread sums four columns of a row over the splits, or, where the
// tile has fewer of those than there are threads, over every `ways`-th split, and the ways
// meet in LDS. Always in the same order. (A thread that walked all splits of a short tile by
// itself: 45 us behind 128 splits of one sequence of 32768 keys, 4 heads.)
template <typename T, typename C, int D, int ROWS>
__global__ void __launch_bounds__(256)
paged_join_kernel(PagedParams<T, C> p) {
  __shared__ float s_w[kJoinWeights];
  __shared__ f32x4 s_o[256];
  const int hk = blockIdx.x % p.at.kv_heads, slot = blockIdx.x / p.at.kv_heads;
  const RowTile rt = RowTile::template at<ROWS>(p, slot);
  if (rt.rows <= 0) return;
  const PageSpan span(rt.position(0), rt.position(rt.rows - 1), rt.length, p.window, p.sinks);
  const int splits = max(1, min(p.splits, (span.tiles + p.split_tiles - 1) / p.split_tiles));
  const Parts<ROWS, D, PagedParams<T, C>> parts(p, slot, hk, 0);  // (a tile's splits are neighbours)
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int row = wave; row < rt.rows; row += 4) {
    float top = -INFINITY, sum = 0.f;
    for (int i = lane; i < splits; i += 64) top = fmaxf(top, parts.ml[2 * (i * ROWS + row)]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    auto weight = [&](int i) { return exp2_fast(parts.ml[2 * (i * ROWS + row)] - top); };
    for (int i = lane; i < splits; i += 64) sum += weight(i) * parts.ml[2 * (i * ROWS + row) + 1];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing: 0
    for (int i = lane; i < splits; i += 64) s_w[row * splits + i] = weight(i) * inv;
  }
  __syncthreads();
  const int units = rt.rows * (D / 4);
  int ways = 1;
  while (2 * ways * units <= 256 && 2 * ways <= splits) ways *= 2;
  for (int u0 = 0; u0 < units; u0 += 256 / ways) {
    const int way = (int)threadIdx.x / (256 / ways), u = u0 + (int)threadIdx.x % (256 / ways);
    const int row = u / (D / 4), col = 4 * (u % (D / 4));
    f32x4 o = zero4();
    if (u < units) {
#pragma unroll 4
      for (int i = way; i < splits; i += ways)
        o += s_w[row * splits + i] * *reinterpret_cast<const f32x4*>(parts.out + (long)(i * ROWS + row) * D + col);
    }
    if (ways > 1) {  // (then this is the only round: units fit 256 / ways threads)
      s_o[threadIdx.x] = o;
      __syncthreads();
      for (int w = 1; w < ways && way == 0; ++w) o += s_o[w * (256 / ways) + threadIdx.x];
    }
    if (way == 0 && u < units)
      *reinterpret_cast<V4<T>*>(p.out + rt.offset(row, hk, p.heads, D) + col) = cvt4<T>(o);
  }
}

template <typename T, typename C, int D, int ROWS>
hipError_t join(const PagedParams<T, C>& p, hipStream_t stream) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  hipLaunchKernelGGL((paged_join_kernel<T, C, D, ROWS>), dim3(p.slots * p.at.kv_heads), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

template <typename T, typename C, int D>
hipError_t launch_paged_attention(const PagedParams<T, C>& p, int rows, hipStream_t stream) {
  const dim3 grid(p.slots * p.at.kv_heads, p.splits);
  if (rows == 128) {
    hipLaunchKernelGGL((paged_chunk_kernel<T, C, D, 4>), grid, dim3(256), 0, stream, p);
    return join<T, C, D, 128>(p, stream);
  }
  if (rows == 64) {
    hipLaunchKernelGGL((paged_chunk_kernel<T, C, D, 2>), grid, dim3(256), 0, stream, p);
    return join<T, C, D, 64>(p, stream);
  }
  constexpr int kWaves = D == 64 ? 8 : D == 128 ? 4 : 2;
  hipLaunchKernelGGL((paged_token_kernel<T, C, D, kWaves>), grid, dim3(64 * kWaves), 0, stream, p);
  return join<T, C, D, kTokenRows>(p, stream);
}

#define FHOG_INST(T, C, D) \
  template hipError_t launch_paged_attention<T, C, D>(const PagedParams<T, C>&, int, hipStream_t);
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
