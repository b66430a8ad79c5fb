// Which blocks of a paged cache a new token attends to (fhog_blocks.h).
//
// A full page has the mean of its keys, m_j = sum over its rows / page_size, summed in 64 bits and rounded to
// fp32 once: sums of 2-byte values are exact there, so a mean does not depend on any order. For a
// token and key/value head, s_j = <sum over its group's queries, m_j> in 64 bits, since a choice has no
// tolerance: fp32 would choose otherwise wherever two scores are within its rounding. A token at
// position p of pages 0 to p / page_size takes the first `first` and the last `last` of them, and of those
// between the ones with the largest scores, ties to the lowest index; NaN is below every number.
//
// The scores go through memory; then the k-th largest is found digit by digit (eight bits of the
// scores' bits in an order that compares as they do), with a histogram in LDS, and the choice is
// written in the order of the columns.
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

// A token's sequence and the columns it may choose from.
struct TokenBlocks {
  int b, own;         // own: the token's own column, -1 if it sees nothing
  int lo, hi;         // columns [lo, hi) are chosen from by score
  int room;           // how many of them
  template <typename P> __device__ __forceinline__ TokenBlocks(const P& p, int t) {
    const CacheShape& c = p.at;
    b = c.offsets ? last_at_or_before(c.batch, t, [&](int s) { return packed_begin(c, s); }) : t;
    const int begin = packed_begin(c, b), end = c.offsets ? packed_begin(c, b + 1) : b + 1;
    const int pos = max(0, c.lengths[b]) - (end - t);
    own = t < begin || t >= end || pos < 0 ? -1 : pos >> c.page_shift;
    if (own >= c.pages_per_seq) own = -1;  // a length beyond the table
    lo = min(p.first, own + 1);
    hi = max(lo, own + 1 - p.last);
    room = max(0, p.blocks - lo - (own + 1 - hi));
  }
  __device__ __forceinline__ bool by_score() const { return hi - lo > room; }
};

// A score's bits in an order that compares as scores do, NaN lowest.
__device__ __forceinline__ unsigned long sortable(double x) {
  if (!(x == x)) return 0;
  const long bits = __builtin_bit_cast(long, x + 0.);  // (-0 + 0 = 0)
  return (unsigned long)bits ^ (bits < 0 ? ~0ul : 1ul << 63);
}

// The scores of kColumns columns of a token and key/value head; sixteen lanes a column.
constexpr int kColumns = 64;
template <typename T, int D> __global__ void __launch_bounds__(kThreads) block_score_kernel(BlockSelectParams<T> p) {
  constexpr int E = D / 16;
  const CacheShape& c = p.at;
  const int hk = blockIdx.x % c.kv_heads, t = p.token0 + blockIdx.x / c.kv_heads;
  const TokenBlocks tb(p, t);
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
  double* const scores = p.scores + (long)blockIdx.x * c.pages_per_seq;
  for (int col = c0 + way; col < min(c0 + kColumns, tb.hi); col += kThreads / 16) {
    if (col < tb.lo) continue;
    const int page = c.table[(long)tb.b * c.pages_per_seq + col];
    double sum = 0.;
    if ((unsigned)page < (unsigned)c.pages) {
      const float* m = p.means + ((long)page * c.kv_heads + hk) * D + lane * 4;
#pragma unroll
      for (int j = 0; j < E; j += 4) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(m + 16 * j);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum = fma(q[j + e], (double)x[e], sum);
      }
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) sum += __shfl_xor(sum, d, 64);
    } else {
      sum = NAN;
    }
    if (lane == 0) scores[col] = sum;
  }
}

template <typename T> __global__ void __launch_bounds__(kThreads) block_choose_kernel(BlockSelectParams<T> p) {
  __shared__ int hist[256], box[4], found[3];
  const CacheShape& c = p.at;
  const int hk = blockIdx.x % c.kv_heads, t = p.token0 + blockIdx.x / c.kv_heads;
  const TokenBlocks tb(p, t);
  int* const out = p.chosen + ((long)t * c.kv_heads + hk) * p.blocks;
  const int count = min(p.blocks, tb.own + 1);
  for (int i = threadIdx.x; i < p.blocks; i += kThreads)
    if (!tb.by_score() || i < tb.lo || i >= tb.lo + tb.room) {
      const int behind = count - i;  // (the last ones end with the token's own)
      out[i] = i >= count ? -1 : i < tb.lo || !tb.by_score() ? i : tb.own + 1 - behind;
    }
  if (!tb.by_score() || tb.room == 0) return;
  const double* const scores = p.scores + (long)blockIdx.x * c.pages_per_seq;
  unsigned long prefix = 0, mask = 0;
  int left = tb.room;
  for (int shift = 56; shift >= 0; shift -= 8) {
    hist[threadIdx.x] = 0;
    __syncthreads();
    for (int col = tb.lo + (int)threadIdx.x; col < tb.hi; col += kThreads) {
      const unsigned long key = sortable(scores[col]);
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
    const unsigned long key = col < tb.hi ? sortable(scores[col]) & mask : 0;
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

template <typename T, int D> hipError_t launch_block_select(const BlockSelectParams<T>& p_, hipStream_t stream) {
  BlockSelectParams<T> p = p_;
  const int slab = p.tokens;
  const unsigned columns = (p.at.pages_per_seq + kColumns - 1) / kColumns;
  for (p.token0 = 0; p.token0 < p.at.total; p.token0 += slab) {
    p.tokens = p.at.total - p.token0 < slab ? p.at.total - p.token0 : slab;
    const unsigned rows = (unsigned)p.tokens * p.at.kv_heads;
    hipLaunchKernelGGL((block_score_kernel<T, D>), dim3(rows, columns), dim3(kThreads), 0, stream, p);
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
  template hipError_t launch_block_select<__bf16, D>(const BlockSelectParams<__bf16>&, hipStream_t);    \
  template hipError_t launch_block_select<_Float16, D>(const BlockSelectParams<_Float16>&, hipStream_t);
FHOG_INST(64)
FHOG_INST(128)
FHOG_INST(256)
#undef FHOG_INST

}  // namespace fhog
