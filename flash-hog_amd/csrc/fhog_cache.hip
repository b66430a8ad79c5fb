// Writing new keys and values into a paged cache, quantised on the way where it holds e4m3,
// and reading sequences back as dense tensors (fhog_paged.h).
//
// e4m3: the scale of a row is the smallest power of two 2^e with which its largest finite
// magnitude stays within 448 = 1.75 2^8, from the magnitude's own exponent; a power of two
// costs a floating format no precision, divides exactly, and is a byte. Values are then
// rounded to nearest, ties to even, by the hardware; a NaN or an infinity becomes NaN and
// leaves the rest of its row alone.
//
// Both kernels move each byte once and hold no state: bound by memory, and for a token or
// two by their launch. A thread takes eight elements of a row.
#include "fhog_paged.h"

namespace fhog {

namespace {

constexpr int kThreads = 256;

// e8m0 code of the scale of a row whose largest finite magnitude is amax.
__device__ __forceinline__ uint32_t scale_code(float amax) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, amax);
  const int code = (int)(bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000);  // 1.75 = 1.11b
  return (uint32_t)max(code, 1);
}

// The e4m3 codes of eight elements of a row and the row's scale code; `lanes` neighbouring
// lanes hold a row.
template <typename T> __device__ __forceinline__ u32x2 quantise8(V8<T> x, int lanes, uint32_t& code) {
  float f[8], amax = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    f[e] = (float)x[e];
    const float a = fabsf(f[e]);
    amax = fmaxf(amax, a < INFINITY ? a : 0.f);  // (false for NaN too)
  }
  for (int d = 1; d < lanes; d <<= 1) amax = fmaxf(amax, __shfl_xor(amax, d, 64));
  code = scale_code(amax);
  const float inv = scale_of(254 - code);  // 2^(127 - code), exact
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = fabsf(f[e]) < INFINITY ? f[e] * inv : NAN;
  u32x2 y;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * h], f[4 * h + 1], 0, false);
    y[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * h + 2], f[4 * h + 3], w, true);
  }
  return y;
}

// A workgroup takes HEADS heads of kRows packed rows: it reads whole lines at a stride, and what it
// writes, neighbouring rows of a head's page and their scales, is contiguous. The rows are
// loaded before their places are looked up, four dependent loads that four heads share where
// there are many rows. Four prompts of up to 8192 tokens, 16 heads, D = 64, e4m3: 47.8 us
// with neighbouring threads on one row's heads, 43.8 with a head a workgroup, 40.8 with four.
template <typename T, typename C, int D, int HEADS>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(CacheWriteParams<T, C> p) {
  constexpr int kLanes = D / 8, kRows = kThreads / kLanes;
  const CacheShape& c = p.at;
  const int groups = (c.kv_heads + HEADS - 1) / HEADS;
  const int col = 8 * (int)(threadIdx.x % kLanes), hk0 = (int)(blockIdx.x % groups) * HEADS;
  const long token = (long)(blockIdx.x / groups) * kRows + threadIdx.x / kLanes;
  // (all lanes of a row take the same way, so quantise8's shuffles find each other)
  if (token >= c.total) return;
  const int heads = min(HEADS, c.kv_heads - hk0);
  V8<T> k[HEADS], v[HEADS];
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    const long from = (token * c.kv_heads + hk0 + min(h, heads - 1)) * D + col;
    k[h] = *reinterpret_cast<const V8<T>*>(p.k + from);
    v[h] = *reinterpret_cast<const V8<T>*>(p.v + from);
  }
  const int t = (int)token;
  const int b = c.offsets ? last_at_or_before(c.batch, t, [&](int s) { return packed_begin(c, s); }) : t;
  const int begin = packed_begin(c, b), end = c.offsets ? packed_begin(c, b + 1) : b + 1;
  if (t < begin || t >= end) return;  // behind the last sequence
  const int pos = max(c.lengths[b], 0) - (end - t);
  if (pos < 0 || (pos >> c.page_shift) >= c.pages_per_seq) return;
  const int page = c.table[(long)b * c.pages_per_seq + (pos >> c.page_shift)];
  if ((unsigned)page >= (unsigned)c.pages) return;
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    if (h >= heads) break;
    const long line = (((long)page * c.kv_heads + hk0 + h) << c.page_shift) + (pos & ((1 << c.page_shift) - 1));
    const long to = line * D + col;
    if constexpr (sizeof(C) == 1) {
      uint32_t kc, vc;
      const u32x2 kq = quantise8<T>(k[h], kLanes, kc), vq = quantise8<T>(v[h], kLanes, vc);
      *reinterpret_cast<u32x2*>(p.k_cache + to) = kq;
      *reinterpret_cast<u32x2*>(p.v_cache + to) = vq;
      if (col == 0) {
        p.k_scale[line] = (uint8_t)kc;
        p.v_scale[line] = (uint8_t)vc;
      }
    } else {
      *reinterpret_cast<V8<T>*>(p.k_cache + to) = k[h];
      *reinterpret_cast<V8<T>*>(p.v_cache + to) = v[h];
    }
  }
}

template <typename T, typename C, int D>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(CacheReadParams<T, C> p) {
  constexpr int kLanes = D / 8;
  const CacheShape& c = p.at;
  const long i = (long)blockIdx.x * kThreads + threadIdx.x;  // (sequence, position, kv_head, eight columns)
  const int col = 8 * (int)(i % kLanes), hk = (int)(i / kLanes % c.kv_heads);
  const long token = i / kLanes / c.kv_heads;
  if (token >= (long)c.batch * p.max_length) return;
  const int b = (int)(token / p.max_length), pos = (int)(token % p.max_length);
  V8<T> k = zero8<T>(), v = zero8<T>();
  if (pos < c.lengths[b]) {
    const int at = pos >> c.page_shift;
    const int page = at < c.pages_per_seq ? c.table[(long)b * c.pages_per_seq + at] : -1;
    if ((unsigned)page < (unsigned)c.pages) {
      const long line = (((long)page * c.kv_heads + hk) << c.page_shift) + (pos & ((1 << c.page_shift) - 1));
      const long from = line * D + col;
      if constexpr (sizeof(C) == 1) {
        const u32x2 kq = *reinterpret_cast<const u32x2*>(p.cache.k + from);
        const u32x2 vq = *reinterpret_cast<const u32x2*>(p.cache.v + from);
        const float ks = scale_of(p.cache.k_scale[line]), vs = scale_of(p.cache.v_scale[line]);
        k = __builtin_shufflevector(dequantise4<T>(kq[0], ks), dequantise4<T>(kq[1], ks), 0, 1, 2, 3, 4, 5, 6, 7);
        v = __builtin_shufflevector(dequantise4<T>(vq[0], vs), dequantise4<T>(vq[1], vs), 0, 1, 2, 3, 4, 5, 6, 7);
      } else {
        k = *reinterpret_cast<const V8<T>*>(p.cache.k + from);
        v = *reinterpret_cast<const V8<T>*>(p.cache.v + from);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) k[e] = v[e] = (T)NAN;
    }
  }
  const long to = (token * c.kv_heads + hk) * D + col;
  *reinterpret_cast<V8<T>*>(p.k + to) = k;
  *reinterpret_cast<V8<T>*>(p.v + to) = v;
}

}  // namespace

template <typename T, typename C, int D>
hipError_t launch_cache_write(const CacheWriteParams<T, C>& p, hipStream_t stream) {
  constexpr int kRows = kThreads / (D / 8);
  const long blocks = ((long)p.at.total + kRows - 1) / kRows;
  const int groups = (p.at.kv_heads + 3) / 4;
  if (blocks * groups >= 1024)
    hipLaunchKernelGGL((cache_write_kernel<T, C, D, 4>), dim3((unsigned)(blocks * groups)), dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((cache_write_kernel<T, C, D, 1>), dim3((unsigned)(blocks * p.at.kv_heads)), dim3(kThreads), 0,
                       stream, p);
  return hipGetLastError();
}

template <typename T, typename C, int D>
hipError_t launch_cache_read(const CacheReadParams<T, C>& p, hipStream_t stream) {
  const long threads = (long)p.at.batch * p.max_length * p.at.kv_heads * (D / 8);
  hipLaunchKernelGGL((cache_read_kernel<T, C, D>), dim3((unsigned)((threads + kThreads - 1) / kThreads)),
                     dim3(kThreads), 0, stream, p);
  return hipGetLastError();
}

#define FHOG_INST(T, C, D)                                                              \
  template hipError_t launch_cache_write<T, C, D>(const CacheWriteParams<T, C>&, hipStream_t); \
  template hipError_t launch_cache_read<T, C, D>(const CacheReadParams<T, C>&, hipStream_t);
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
