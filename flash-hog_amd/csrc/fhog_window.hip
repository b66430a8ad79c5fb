// Launches of the windowed attention (MASK = kWindow): the forward, the first backward
// and the double backward take the kernels of the other masks in their window mode.
//
// A sink is seen by every query behind it, an ordinary key by `window` of them. One
// workgroup per key block would give the block with the sinks n_q queries where the others
// have window + 64: at N = 16384 with a window of 1024 fifteen times their work, the whole
// launch's length. So the queries that see a sink as a sink only are dealt to further
// workgroups in chunks about as long as an ordinary block's share (SinkGrid). Each writes its
// part of the sinks' rows in fp32, and sink_join_kernel adds a row's parts, always in the
// same order (no atomics: repeated calls give the same bits), and rounds the sum once.
#include "fhog_device.h"
#include "fhog_params.h"

namespace fhog {

namespace {

// dk and dv of the sinks from their parts, four columns a thread. Reads (1 + chunks) fp32
// rows for each row it writes, a few hundred KB in all: bound by its launch.
template <typename T, int D>
__global__ void __launch_bounds__(256)
sink_join_kernel(const float* parts, T* dk, T* dv, int pairs, int kv_heads, int nk, int sinks, int count) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;  // (batch, kv_head, sink, dV or dK, column / 4)
  constexpr int kCols = D / 4;
  const long rows = 2l * pairs * sinks;
  if (i >= rows * kCols) return;
  const long row = i / kCols;
  const int col = 4 * (int)(i % kCols);
  f32x4 sum = zero4();
#pragma unroll 8
  for (int c = 0; c < count; ++c) sum += *reinterpret_cast<const f32x4*>(parts + (c * rows + row) * D + col);
  const int key = (int)(row / 2 % sinks), bh = (int)(row / 2 / sinks);
  const int b = bh / kv_heads, hk = bh % kv_heads;
  T* dst = (row & 1 ? dk : dv) + (((long)b * nk + key) * kv_heads + hk) * D + col;
  *reinterpret_cast<V4<T>*>(dst) = cvt4<T>(sum);
}

template <typename T, int D, typename P>
hipError_t join(const P& p, T* dk, T* dv, hipStream_t stream) {
  if (p.sink.chunks == 0) return hipSuccess;
  const int pairs = p.batch * p.kv_heads, sinks = p.sinks < p.nk ? p.sinks : p.nk;
  const long threads = 2l * pairs * sinks * (D / 4);
  hipLaunchKernelGGL((sink_join_kernel<T, D>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream,
                     p.sink_parts, dk, dv, pairs, p.kv_heads, p.nk, sinks, 1 + p.sink.chunks);
  return hipGetLastError();
}

}  // namespace

// dK and dV: FLASH_HOG_BWD = few (rows of up to 256 bytes) or pair, or the rules of fhog_grid.h.
template <typename T, int D> hipError_t launch_window_dkdv(const BwdParams<T>& p, hipStream_t stream) {
  if constexpr (kFewServes<T, D>) {
    if (p.sink.apart && p.sink.chunks > 0) {
      const hipError_t e = launch_few_dkdv<T, D>(p, true, stream);
      if (e != hipSuccess) return e;
    }
  }
  const BwdParams<T> own = own_launch(p);
  if constexpr (kFewServes<T, D>) {
    if (window_few_selected(std::getenv("FLASH_HOG_BWD"), FewKernel::kDkdv, key_grid<kWindow>(own, 32), D,
                            (int)sizeof(T)))
      return launch_few_dkdv<T, D>(own, false, stream);
  }
  return launch_bwd_pair<T, D, kWindow>(own, stream);
}

template <typename T, int D> hipError_t launch_window_bwd(const BwdParams<T>& p, hipStream_t stream) {
  hipError_t e = launch_window_dq<T, D>(p, stream);
  if (e == hipSuccess) e = launch_window_dkdv<T, D>(p, stream);
  return e == hipSuccess ? join<T, D>(p, p.dk, p.dv, stream) : e;
}

template <typename T, int D> hipError_t launch_window_bwdbwd(const BwdBwdParams<T>& p, hipStream_t stream) {
  hipError_t e;
  if constexpr (sizeof(T) == 4)
    e = launch_bwdbwd_stage1_qpair<D, kWindow>(p, stream);
  else if constexpr (D == 128)
    e = launch_bwdbwd_stage1_fused_pair<T, kWindow>(p, stream);
  else
    e = launch_bwdbwd_stage1_fused<T, D, kWindow>(p, stream);
  if (e == hipSuccess) e = launch_window_stage2<T, D>(p, stream);
  return e == hipSuccess ? join<T, D>(p, p.dk2, p.dv2, stream) : e;
}

#define FHOG_INST(T, D)                                                         \
  template hipError_t launch_window_bwd<T, D>(const BwdParams<T>&, hipStream_t); \
  template hipError_t launch_window_bwdbwd<T, D>(const BwdBwdParams<T>&, hipStream_t);
FHOG_INST(__bf16, 64)
FHOG_INST(__bf16, 128)
FHOG_INST(__bf16, 256)
FHOG_INST(_Float16, 64)
FHOG_INST(_Float16, 128)
FHOG_INST(_Float16, 256)
FHOG_INST(float, 64)
FHOG_INST(float, 128)
#undef FHOG_INST

}  // namespace fhog
