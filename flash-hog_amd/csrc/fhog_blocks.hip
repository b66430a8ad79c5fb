// Attention of new tokens over chosen blocks of a paged cache (fhog_blocks.h): each packed token and key/value
// head has a list of columns of its sequence's page table, and its queries see the keys of these pages up to
// the token's own position.
//
// block_token_kernel: as paged_token_kernel, with the list in place of the sequence's pages. The rows of a
// workgroup are one token's, so masks are a number of visible rows a block, the same for all; a half tile
// of 16 keys never leaves a page, and halves that show nothing are not read. Scores, statistics and
// running outputs are fp32; a probability enters the second product in T, half a step of rounding a term,
// as in the other paged kernels.
#include "fhog_blocks.h"

namespace fhog {

namespace {

constexpr float kBound = 256.f;  // bound on an unnormalised probability
constexpr int kRows = 16;

// A slot's token, and its rows of the token's group.
struct TokenRows {
  int t, row0, rows, group;
  int b, pos;
  bool there, beyond;  // whether the token is a sequence's; whether its length is beyond the table
  template <typename P> __device__ __forceinline__ TokenRows(const P& p, int slot) {
    const CacheShape& c = p.at;
    group = p.heads / c.kv_heads;
    const int tiles = (group + kRows - 1) / kRows;
    t = slot / tiles;
    row0 = slot % tiles * kRows;
    rows = min(kRows, group - row0);
    b = c.offsets ? last_at_or_before(c.batch, t, [&](int s) { return packed_begin(c, s); }) : t;
    const int begin = packed_begin(c, b), end = c.offsets ? packed_begin(c, b + 1) : b + 1;
    there = t >= begin && t < end;
    const int length = max(0, c.lengths[b]);
    beyond = length > (long)c.pages_per_seq << c.page_shift;
    pos = length - (end - t);
  }
  __device__ __forceinline__ long offset(int r, int hk, int heads, int d) const {
    return ((long)t * heads + hk * group + row0 + r) * d;
  }
};

// A block's page and how many of its rows the token sees.
struct BlockEntry {
  int page, rows;
};

template <typename T, typename C, int D, int kWaves>
__global__ void __launch_bounds__(64 * kWaves) block_token_kernel(BlockParams<T, C> p) {
  constexpr int KS = D / 32, DB = D / 16;
  typedef KeyPieces<T, C, D> Keys;
  constexpr bool kDirect = Keys::kQuantised;
  typedef PageTile<T, C, D, 64, D == 64 ? kSwzRows : kSwzWide, kDirect ? 1 : 2> Tile;
  constexpr int kWaveLds = (kDirect ? 1 : 2) * Tile::kTileBytes;
  __shared__ __attribute__((aligned(1024))) char s_kv[kWaves * kWaveLds];
  __shared__ float s_ml[kWaves][kRows][2];
  __shared__ BlockEntry s_entry[kSplitBlocks];
  __shared__ int s_bad;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const CacheShape& c = p.at;
  const int hk = blockIdx.x % c.kv_heads, slot = blockIdx.x / c.kv_heads, split = blockIdx.y;
  const TokenRows tr(p, p.slot0 + slot);
  if (!tr.there) {
    if (p.clear_rest && split == 0)
      for (int i = threadIdx.x; i < tr.rows * (D / 8); i += 64 * kWaves)
        *reinterpret_cast<V8<T>*>(p.out + tr.offset(0, hk, p.heads, D) + 8 * i) = zero8<T>();
    return;
  }
  const int page_rows = 1 << c.page_shift;
  const int tiles = (int)(((long)p.blocks * page_rows + 31) / 32);
  const int t0 = split * p.split_tiles, t1 = min(tiles, t0 + p.split_tiles);

  // This split's blocks.
  const int e0 = (int)((32l * t0) >> c.page_shift);
  const int e1 = (int)min((long)p.blocks, (32l * t1 + page_rows - 1) >> c.page_shift);
  if (threadIdx.x == 0) s_bad = 0;
  __syncthreads();
  for (int i = e0 + threadIdx.x; i < e1; i += 64 * kWaves) {
    const int col = p.chosen[((long)tr.t * c.kv_heads + hk) * p.blocks + i];
    BlockEntry e{0, 0};
    if (col >= 0 && col < c.pages_per_seq) {
      const long seen = (long)tr.pos + 1 - ((long)col << c.page_shift);
      e.rows = (int)(seen < 0 ? 0 : seen < page_rows ? seen : page_rows);
      if (e.rows > 0) e.page = c.table[(long)tr.b * c.pages_per_seq + col];
      if ((unsigned)e.page >= (unsigned)c.pages) {
        e.page = 0;
        s_bad = 1;
      }
    }
    s_entry[i - e0] = e;
  }

  const int r = min(n, tr.rows - 1);
  const bool negate = p.scale < 0.f;  // applied as |scale| to -q (negation is exact)
  V8<T> qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    qf[ks] = *reinterpret_cast<const V8<T>*>(p.q + tr.offset(r, hk, p.heads, D) +
                                             (kDirect ? Keys::column(ks, g) : 32 * ks + 8 * g));
    if (negate) qf[ks] = -qf[ks];
  }
  const float c2 = fabsf(p.scale) * kLog2e;
  __syncthreads();

  std::conditional_t<D == 64, SwzFrags16<T, D>, WideFrags16<T, D>> fr;
  fr.init(lane);
  const uint32_t lds = lds_base_u32(s_kv) + wave * kWaveLds;
  float m = -1e30f, lpart = 0.f;
  f32x4 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) acc[db] = zero4();

  // Rows of a tile's halves that are seen, and where they lie; the same in all lanes.
  struct Place {
    HalfRows at;
    int seen[2];
  };
  auto place = [&](int t) {
    Place x;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long key = 32l * t + 16 * h;
      const int e = (int)(key >> c.page_shift), r0 = (int)(key & (page_rows - 1));
      int page = 0, rows = 0;
      if (e < e1) {
        page = __builtin_amdgcn_readfirstlane(s_entry[e - e0].page);
        rows = __builtin_amdgcn_readfirstlane(s_entry[e - e0].rows);
      }
      x.seen[h] = min(16, max(0, rows - r0));
      x.at.line[h] = (((long)page * c.kv_heads + hk) << c.page_shift) + r0;
      x.at.last[h] = x.seen[h] - 1;
    }
    if (x.seen[0] == 0) x.at.line[0] = x.at.line[1], x.at.last[0] = x.at.last[1];
    if (x.seen[1] == 0) x.at.line[1] = x.at.line[0], x.at.last[1] = x.at.last[0];
    return x;
  };
  Keys keys;
  Tile tile;
  Place now, next;
  // This wave's first tile from t on that shows something; fetched.
  auto fetch = [&](int t) {
    for (; t < t1; t += kWaves) {
      next = place(t);
      if (next.seen[0] + next.seen[1] > 0) break;
    }
    if (t < t1) {
      if constexpr (kDirect) keys.fetch(p.cache, next.at, n, g);
      tile.fetch(p.cache, next.at, lane);
    }
    return t;
  };
  for (int t = fetch(t0 + wave); t < t1;) {
    now = next;
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
    t = fetch(t + kWaves);
    if constexpr (!kDirect) scores([&](int kb, int ks) { return fr.rowf(lds, 0, kb, ks); });
    if (now.seen[0] < 16 || now.seen[1] < 16) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (4 * g + (e & 3) >= now.seen[e >> 2]) S[e >> 2][e & 3] = -INFINITY;
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

  // The waves' outputs meet in LDS, in place of the tiles: (wave, column, row).
  if (s_bad || tr.beyond) lpart = NAN;
  const float l = group4_sum(lpart);
  __syncthreads();
  float* so = reinterpret_cast<float*>(s_kv);
  static_assert(kWaves * kRows * D * (int)sizeof(float) <= kWaves * kWaveLds, "the join reuses the tiles");
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i) so[(wave * D + 16 * db + 4 * g + i) * kRows + n] = acc[db][i];
  if (g == 0) {
    s_ml[wave][n][0] = m;
    s_ml[wave][n][1] = l;
  }
  __syncthreads();
  const long part = ((long)slot * c.kv_heads + hk) * p.splits + split, parts = (long)p.slots * c.kv_heads * p.splits;
  float* const part_out = p.parts + part * kRows * D;
  float* const part_ml = p.parts + parts * kRows * D + part * kRows * 2;
  for (int i = threadIdx.x; i < kRows * (D / 4); i += 64 * kWaves) {
    const int row = i / (D / 4), col = 4 * (i % (D / 4));
    if (row >= tr.rows) break;
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
      for (int j = 0; j < 4; ++j) o[j] += f * so[(w * D + col + j) * kRows + row];
    }
    if (p.splits > 1) {
      *reinterpret_cast<f32x4*>(part_out + row * D + col) = o;
      if (col == 0) {
        part_ml[2 * row] = top;
        part_ml[2 * row + 1] = sum;
      }
    } else {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing: 0
      *reinterpret_cast<V4<T>*>(p.out + tr.offset(row, hk, p.heads, D) + col) = cvt4<T>(o * inv);
    }
  }
}

// Joins the splits, in order: a workgroup a slot and key/value head. The rows' weights first, then four
// columns a thread.
template <typename T, typename C, int D> __global__ void __launch_bounds__(256) block_join_kernel(BlockParams<T, C> p) {
  __shared__ float s_w[kJoinWeights];
  const CacheShape& c = p.at;
  const int hk = blockIdx.x % c.kv_heads, slot = blockIdx.x / c.kv_heads;
  const TokenRows tr(p, p.slot0 + slot);
  if (!tr.there) return;
  const long part = ((long)slot * c.kv_heads + hk) * p.splits, parts = (long)p.slots * c.kv_heads * p.splits;
  const float* const part_out = p.parts + part * kRows * D;
  const float* const part_ml = p.parts + parts * kRows * D + part * kRows * 2;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int row = wave; row < tr.rows; row += 4) {
    float top = -INFINITY, sum = 0.f;
    for (int i = lane; i < p.splits; i += 64) top = fmaxf(top, part_ml[2 * (i * kRows + row)]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
    auto weight = [&](int i) { return exp2_fast(part_ml[2 * (i * kRows + row)] - top); };
    for (int i = lane; i < p.splits; i += 64) sum += weight(i) * part_ml[2 * (i * kRows + row) + 1];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    for (int i = lane; i < p.splits; i += 64) s_w[row * p.splits + i] = weight(i) * inv;
  }
  __syncthreads();
  for (int u = threadIdx.x; u < tr.rows * (D / 4); u += 256) {
    const int row = u / (D / 4), col = 4 * (u % (D / 4));
    f32x4 o = zero4();
    for (int i = 0; i < p.splits; ++i)
      o += s_w[row * p.splits + i] * *reinterpret_cast<const f32x4*>(part_out + (long)(i * kRows + row) * D + col);
    *reinterpret_cast<V4<T>*>(p.out + tr.offset(row, hk, p.heads, D) + col) = cvt4<T>(o);
  }
}

}  // namespace

template <typename T, typename C, int D>
hipError_t launch_block_attention(const BlockParams<T, C>& p_, int slab, hipStream_t stream) {
  constexpr int kWaves = D == 64 ? 8 : D == 128 ? 4 : 2;
  BlockParams<T, C> p = p_;
  for (p.slot0 = 0; p.slot0 < p_.slots; p.slot0 += slab) {
    p.slots = p_.slots - p.slot0 < slab ? p_.slots - p.slot0 : slab;
    const dim3 grid(p.slots * p.at.kv_heads, p.splits);
    hipLaunchKernelGGL((block_token_kernel<T, C, D, kWaves>), grid, dim3(64 * kWaves), 0, stream, p);
    if (p.splits > 1) hipLaunchKernelGGL((block_join_kernel<T, C, D>), dim3(grid.x), dim3(256), 0, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

#define FHOG_INST(T, C, D) template hipError_t launch_block_attention<T, C, D>(const BlockParams<T, C>&, int, hipStream_t);
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
