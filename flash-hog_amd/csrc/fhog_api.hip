// C-ABI entry points: argument validation and dispatch to the templated
// launchers. Error reporting follows the reference's FFI handler
// (flash_hog/csrc/tk_bwdbwd/ffi.cu:35-39, 74-76): invalid shapes are rejected
// before anything is enqueued, launch failures are reported with the runtime's
// message. Messages are kept per thread; there is no other global state.
#include <stdint.h>
#include <stdio.h>
#include <stdarg.h>
#include <string.h>

#include <atomic>
#include <mutex>

#include "flash_hog.h"
#include "fhog_params.h"
#include "fhog_paged.h"
#include "fhog_pages.h"
#include "fhog_blocks.h"
#include "fhog_rotary.h"

namespace {

thread_local char g_last_error[512] = "";

int fail(int status, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
  return status;
}

int ok() {
  g_last_error[0] = '\0';
  return FHOG_OK;
}

// Tensors are read with 16-byte vector loads; fp32 row statistics with scalar loads.
bool aligned(const void* p, uintptr_t bytes) {
  return p != nullptr && (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

struct Shape {
  int batch, n_q, n_k, heads, kv_heads, head_dim, dtype, causal;
  float scale;
  // Key j is visible to query i iff j <= i + coff (causal kernels only).
  int coff() const { return causal == FHOG_CAUSAL_BOTTOM_RIGHT ? n_k - n_q : 0; }
};

int check_shape(const Shape& s, const char* who) {
  if (!(s.scale == s.scale) || s.scale - s.scale != 0.0f)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: scale must be finite", who);
  // With scale 0 every logit is 0 and masked ones are -inf * 0; the kernels
  // also divide by the scale. Any other finite scale, negative included, works.
  if (s.scale == 0.0f) return fail(FHOG_ERR_UNSUPPORTED, "%s: scale must be nonzero", who);
  if (s.causal != FHOG_CAUSAL_NONE && s.causal != FHOG_CAUSAL_TOP_LEFT && s.causal != FHOG_CAUSAL_BOTTOM_RIGHT)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: causal must be 0 (none), 1 (top-left) or 2 (bottom-right), got %d",
                who, s.causal);
  if (s.batch < 1 || s.n_q < 1 || s.n_k < 1 || s.heads < 1 || s.kv_heads < 1)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: sizes must be >= 1 (batch=%d n_q=%d n_k=%d heads=%d kv_heads=%d)",
                who, s.batch, s.n_q, s.n_k, s.heads, s.kv_heads);
  if (s.dtype != FHOG_DTYPE_F32 && s.dtype != FHOG_DTYPE_F16 && s.dtype != FHOG_DTYPE_BF16)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", who, s.dtype);
  if (s.head_dim < 1)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: head_dim must be >= 1, got %d", who, s.head_dim);
  if (s.heads % s.kv_heads != 0)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: heads (%d) must be a multiple of kv_heads (%d)", who, s.heads,
                s.kv_heads);
  if (s.dtype == FHOG_DTYPE_F32 && s.head_dim != 64 && s.head_dim != 128)
    return fail(FHOG_ERR_UNSUPPORTED, "%s: fp32 head_dim must be 64 or 128, got %d", who, s.head_dim);
  if (s.head_dim != 64 && s.head_dim != 128 && s.head_dim != 256)
    return fail(FHOG_ERR_UNSUPPORTED, "%s: head_dim must be 64, 128 or 256, got %d", who, s.head_dim);
  const long long rows = (long long)s.batch * s.heads * (s.n_q > s.n_k ? s.n_q : s.n_k);
  if (rows * s.head_dim >= (1ll << 40) || (long long)s.batch * s.heads * ((s.n_q > s.n_k ? s.n_q : s.n_k) + 31) / 32 >= (1ll << 31))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: problem too large", who);
  return FHOG_OK;
}

int check_ptrs(const char* who, std::initializer_list<std::pair<const char*, const void*>> tensors,
               std::initializer_list<std::pair<const char*, const void*>> row_stats) {
  for (const auto& p : tensors)
    if (!aligned(p.second, 16))
      return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: %s is null or not 16-byte aligned", who, p.first);
  for (const auto& p : row_stats)
    if (!aligned(p.second, 4))
      return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: %s is null or not 4-byte aligned", who, p.first);
  return FHOG_OK;
}

int launch_status(hipError_t e, const char* who) {
  if (e != hipSuccess) return fail(FHOG_ERR_LAUNCH, "%s: %s", who, hipGetErrorString(e));
  return ok();
}

// Calls f.template operator()<T, D, CAUSAL>() for the runtime (dtype, head_dim, causal).
template <typename F>
hipError_t dispatch(int dtype, int head_dim, bool causal, F&& f) {
#define FHOG_CASE(T, D)                                          \
  return causal ? f.template operator()<T, D, true>() : f.template operator()<T, D, false>();
  if (dtype == FHOG_DTYPE_BF16) {
    if (head_dim == 64) { FHOG_CASE(__bf16, 64) }
    if (head_dim == 128) { FHOG_CASE(__bf16, 128) }
    FHOG_CASE(__bf16, 256)
  }
  if (dtype == FHOG_DTYPE_F16) {
    if (head_dim == 64) { FHOG_CASE(_Float16, 64) }
    if (head_dim == 128) { FHOG_CASE(_Float16, 128) }
    FHOG_CASE(_Float16, 256)
  }
  if (head_dim == 64) { FHOG_CASE(float, 64) }
  FHOG_CASE(float, 128)
#undef FHOG_CASE
}

// Calls f.template operator()<T, D>() for the runtime (dtype, head_dim).
template <typename F> hipError_t dispatch(int dtype, int head_dim, F&& f) {
  return dispatch(dtype, head_dim, false, [&]<typename T, int D, bool C>() { return f.template operator()<T, D>(); });
}

// A window of keys and sinks, as the kernels take them: both cut to what the sizes can show.
struct Window {
  int window, sinks;
  fhog::SinkGrid sink;
};

int check_window(const Shape& s, int window, int sinks, Window* w, const char* who) {
  if (int st = check_shape(s, who)) return st;
  if (s.causal == FHOG_CAUSAL_NONE)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: a window needs causal 1 (top-left) or 2 (bottom-right)", who);
  if (window < 1) return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: window must be >= 1, got %d", who, window);
  if (sinks < 0) return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: sinks must be >= 0, got %d", who, sinks);
  const int most = s.n_q > s.n_k ? s.n_q : s.n_k;
  if (most > (1 << 30)) return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: problem too large", who);
  w->window = window < most ? window : most;  // positions are below `most`
  w->sinks = sinks < s.n_k ? sinks : s.n_k;
  const fhog::Mask m{true, s.n_q, s.n_k, s.coff()};
  const int row_bytes = s.head_dim * (s.dtype == FHOG_DTYPE_F32 ? 4 : 2);
  const fhog::SinkChunks c = fhog::sink_chunks(m, w->window, w->sinks, row_bytes, (long)s.batch * s.heads,
                                               (long)s.batch * s.kv_heads);
  w->sink = fhog::SinkGrid{(w->sinks + 31) / 32, c.count, c.step, c.apart};
  const long long groups = ((s.n_k + 31) / 32 + (long long)w->sink.blocks * w->sink.chunks) * s.batch * s.kv_heads;
  if (groups >= (1ll << 31)) return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: problem too large", who);
  return FHOG_OK;
}

size_t sink_parts_bytes(const Shape& s, const Window& w) {
  if (w.sink.chunks == 0) return 0;
  return (size_t)(1 + w.sink.chunks) * s.batch * s.kv_heads * w.sinks * 2 * s.head_dim * sizeof(float);
}

// The workspace of a call that has sinks to join.
int check_workspace(const char* who, const Window& w, const void* workspace) {
  if (w.sink.chunks > 0 && !aligned(workspace, 16))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: workspace is null or not 16-byte aligned", who);
  return FHOG_OK;
}

}  // namespace

namespace {

// What the three paged entry points share. `rows`: the packed rows (attention, write).
struct Paged {
  int batch, rows, heads, kv_heads, head_dim, num_pages, page_size, pages_per_seq, dtype, cache_dtype;
};

constexpr double kMostElements = 32.0 * (1ll << 30);  // of a packed tensor; eight a thread

int check_paged(const Paged& s, const char* who) {
  if (s.batch < 0 || s.rows < 0) return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: sizes must not be negative", who);
  if (s.heads < 1 || s.kv_heads < 1 || s.num_pages < 1 || s.pages_per_seq < 1)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: sizes must be >= 1 (heads=%d kv_heads=%d num_pages=%d pages_per_seq=%d)",
                who, s.heads, s.kv_heads, s.num_pages, s.pages_per_seq);
  if (s.heads % s.kv_heads != 0)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: heads (%d) must be a multiple of kv_heads (%d)", who, s.heads,
                s.kv_heads);
  if (s.page_size < 16 || (s.page_size & (s.page_size - 1)) != 0)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: page_size must be a power of two >= 16, got %d", who, s.page_size);
  if (s.dtype != FHOG_DTYPE_F16 && s.dtype != FHOG_DTYPE_BF16)
    return fail(FHOG_ERR_UNSUPPORTED, "%s: dtype must be bf16 or fp16, got %d", who, s.dtype);
  if (s.cache_dtype != s.dtype && s.cache_dtype != FHOG_DTYPE_E4M3)
    return fail(FHOG_ERR_UNSUPPORTED, "%s: the cache must be of dtype %d or e4m3, got %d", who, s.dtype, s.cache_dtype);
  if (s.head_dim != 64 && s.head_dim != 128 && s.head_dim != 256)
    return fail(FHOG_ERR_UNSUPPORTED, "%s: head_dim must be 64, 128 or 256, got %d", who, s.head_dim);
  // packed (token, head) rows and positions are ints, a launch's threads 32 bits
  if ((long long)s.rows * s.heads >= (1ll << 30) || (double)s.rows * s.heads * s.head_dim >= kMostElements ||
      s.batch >= (1 << 24) ||
      (long long)s.pages_per_seq * s.page_size > (1ll << 30))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: problem too large", who);
  return FHOG_OK;
}

int check_cache(const char* who, const Paged& s, const void* k, const void* v, const void* ks, const void* vs,
                const void* table, const void* lengths) {
  if (int st = check_ptrs(who, {{"k_cache", k}, {"v_cache", v}}, {{"page_table", table}, {"lengths", lengths}}))
    return st;
  if (s.cache_dtype == FHOG_DTYPE_E4M3 && (ks == nullptr || vs == nullptr))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: an e4m3 cache needs k_scale and v_scale", who);
  return FHOG_OK;
}

fhog::CacheShape cache_shape(const Paged& s, const int* table, const int* lengths, const int* offsets) {
  return fhog::CacheShape{table, lengths, offsets, s.batch, s.rows, s.kv_heads, s.num_pages,
                          __builtin_ctz((unsigned)s.page_size), s.pages_per_seq};
}

// Calls f.template operator()<T, C, D>() for the runtime (dtype, cache_dtype, head_dim).
template <typename F> hipError_t dispatch_paged(const Paged& s, F&& f) {
  auto dim = [&]<typename T, typename C>() {
    if (s.head_dim == 64) return f.template operator()<T, C, 64>();
    if (s.head_dim == 128) return f.template operator()<T, C, 128>();
    return f.template operator()<T, C, 256>();
  };
  const bool quantised = s.cache_dtype == FHOG_DTYPE_E4M3;
  if (s.dtype == FHOG_DTYPE_BF16)
    return quantised ? dim.template operator()<__bf16, fhog::e4m3>() : dim.template operator()<__bf16, __bf16>();
  return quantised ? dim.template operator()<_Float16, fhog::e4m3>() : dim.template operator()<_Float16, _Float16>();
}

int compute_units() {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
    return 0;
  return cus;
}

}  // namespace

extern "C" {

int fhog_abi_version(void) { return 103; }

const char* fhog_status_string(int status) {
  switch (status) {
    case FHOG_OK: return "ok";
    case FHOG_ERR_INVALID_ARGUMENT: return "invalid argument";
    case FHOG_ERR_UNSUPPORTED: return "unsupported";
    case FHOG_ERR_LAUNCH: return "kernel launch failed";
    default: return "unknown status";
  }
}

const char* fhog_last_error(void) { return g_last_error; }

int fhog_attention_supported(int device, int batch, int n_q, int n_k, int heads, int kv_heads, int head_dim,
                             int dtype, int causal, float scale) {
  static const char* who = "fhog_attention_supported";
  const Shape s{batch, n_q, n_k, heads, kv_heads, head_dim, dtype, causal, scale};
  if (int st = check_shape(s, who)) return st;
  if (device >= 0) {
    hipDeviceProp_t prop;
    const hipError_t e = hipGetDeviceProperties(&prop, device);
    if (e != hipSuccess)
      return fail(FHOG_ERR_UNSUPPORTED, "%s: no HIP device %d (%s)", who, device, hipGetErrorString(e));
    if (strncmp(prop.gcnArchName, "gfx950", 6) != 0)
      return fail(FHOG_ERR_UNSUPPORTED, "%s: device %d is %s; the kernels are built for gfx950", who, device,
                  prop.gcnArchName);
  }
  return ok();
}

size_t fhog_row_stat_bytes(int batch, int heads, int n_q) {
  if (batch < 1 || heads < 1 || n_q < 1) return 0;
  return (size_t)batch * heads * n_q * sizeof(float);
}

int fhog_attention_fwd(fhog_stream_t stream, const void* q, const void* k, const void* v, void* o, float* lse,
                       int batch, int n_q, int n_k, int heads, int kv_heads, int head_dim, int dtype, int causal,
                       float scale) {
  static const char* who = "fhog_attention_fwd";
  const Shape s{batch, n_q, n_k, heads, kv_heads, head_dim, dtype, causal, scale};
  if (int st = check_shape(s, who)) return st;
  if (int st = check_ptrs(who, {{"q", q}, {"k", k}, {"v", v}, {"o", o}}, {{"lse", lse}})) return st;
  auto run = [&]<typename T, int D, bool C>() {
    fhog::FwdParams<T> p{(const T*)q, (const T*)k, (const T*)v, (T*)o, lse, batch, n_q, n_k, heads, kv_heads,
                         s.coff(), scale};
    return fhog::launch_fwd<T, D, C>(p, (hipStream_t)stream);
  };
  return launch_status(dispatch(dtype, head_dim, causal != 0, run), who);
}

int fhog_attention_bwd(fhog_stream_t stream, const void* q, const void* k, const void* v, const void* o,
                       const void* dout, const float* lse, void* dq, void* dk, void* dv, float* delta, int batch,
                       int n_q, int n_k, int heads, int kv_heads, int head_dim, int dtype, int causal, float scale) {
  static const char* who = "fhog_attention_bwd";
  const Shape s{batch, n_q, n_k, heads, kv_heads, head_dim, dtype, causal, scale};
  if (int st = check_shape(s, who)) return st;
  if (int st = check_ptrs(who, {{"q", q}, {"k", k}, {"v", v}, {"o", o}, {"dout", dout}, {"dq", dq}, {"dk", dk},
                                {"dv", dv}},
                           {{"lse", lse}, {"delta", delta}}))
    return st;
  auto run = [&]<typename T, int D, bool C>() {
    fhog::BwdParams<T> p{(const T*)q, (const T*)k, (const T*)v, (const T*)o, (const T*)dout, lse,
                         (T*)dq, (T*)dk, (T*)dv, delta, batch, n_q, n_k, heads, kv_heads, s.coff(), scale};
    return fhog::launch_bwd<T, D, C>(p, (hipStream_t)stream);
  };
  return launch_status(dispatch(dtype, head_dim, causal != 0, run), who);
}

namespace {

int bwdbwd_impl(const char* who, int stages, fhog_stream_t stream, const void* q, const void* k, const void* v,
                const void* o, const void* dout, const void* ddq, const void* ddk, const void* ddv,
                const float* lse, void* dq2, void* dk2, void* dv2, void* ddo, float* delta, float* ddelta,
                float* bstat, int batch, int n_q, int n_k, int heads, int kv_heads, int head_dim, int dtype,
                int causal, float scale) {
  const Shape s{batch, n_q, n_k, heads, kv_heads, head_dim, dtype, causal, scale};
  if (int st = check_shape(s, who)) return st;
  if (int st = check_ptrs(who, {{"q", q}, {"k", k}, {"v", v}, {"dout", dout}, {"ddq", ddq}, {"ddk", ddk},
                                {"ddv", ddv}},
                           {{"lse", lse}, {"delta", delta}, {"ddelta", ddelta}, {"bstat", bstat}}))
    return st;
  if (stages & 1)
    if (int st = check_ptrs(who, {{"o", o}, {"dq2", dq2}, {"ddo", ddo}}, {})) return st;
  if (stages & 2)
    if (int st = check_ptrs(who, {{"dk2", dk2}, {"dv2", dv2}}, {})) return st;
  auto run = [&]<typename T, int D, bool C>() {
    fhog::BwdBwdParams<T> p{(const T*)q,   (const T*)k,   (const T*)v,   (const T*)o, (const T*)dout,
                            (const T*)ddq, (const T*)ddk, (const T*)ddv, lse,         (T*)dq2,
                            (T*)dk2,       (T*)dv2,       (T*)ddo,       delta,       ddelta,
                            bstat,         batch,         n_q,           n_k,         heads,
                            kv_heads,      s.coff(),      scale};
    return fhog::launch_bwdbwd<T, D, C>(p, (hipStream_t)stream, stages);
  };
  return launch_status(dispatch(dtype, head_dim, causal != 0, run), who);
}

// ---------------------------------------------------------------------------
// Row statistics of fhog_attention_bwdbwd_noalloc: D, dD and B of up to
// kScratchRows (batch, head, query) rows each, in one file-scope device array
// (12 MiB per device, held until the process ends). Every call on a device
// uses that device's copy; the kernels write every row they later read, so
// nothing needs clearing between calls, but two calls that overlap on one
// device race on it.
// ---------------------------------------------------------------------------
constexpr long long kScratchRows = 1ll << 20;
static __device__ __align__(256) float scratch[3 * kScratchRows];

// Device address of `scratch` per device, looked up once per device (with
// that device current) and kept: in host code the array's name is not a
// device address.
constexpr int kMaxDevices = 64;
std::atomic<float*> g_scratch[kMaxDevices];
std::mutex g_scratch_mu;

int scratch_address(const char* who, hipStream_t stream, float** out) {
  int dev = -1;
  hipError_t e = stream ? hipStreamGetDevice(stream, &dev) : hipGetDevice(&dev);
  if (e != hipSuccess) return fail(FHOG_ERR_LAUNCH, "%s: cannot find the stream's device: %s", who, hipGetErrorString(e));
  if (dev < 0 || dev >= kMaxDevices) return fail(FHOG_ERR_UNSUPPORTED, "%s: device %d out of range", who, dev);
  float* ptr = g_scratch[dev].load(std::memory_order_acquire);
  if (ptr == nullptr) {
    std::lock_guard<std::mutex> lock(g_scratch_mu);
    ptr = g_scratch[dev].load(std::memory_order_relaxed);
    if (ptr == nullptr) {
      int cur = -1;
      if ((e = hipGetDevice(&cur)) == hipSuccess && cur != dev) e = hipSetDevice(dev);
      void* addr = nullptr;
      if (e == hipSuccess) e = hipGetSymbolAddress(&addr, HIP_SYMBOL(scratch));
      if (cur >= 0 && cur != dev) {
        const hipError_t back = hipSetDevice(cur);
        if (e == hipSuccess) e = back;
      }
      if (e != hipSuccess || addr == nullptr)
        return fail(FHOG_ERR_LAUNCH, "%s: no address for the static scratch on device %d: %s", who, dev,
                    hipGetErrorString(e));
      ptr = static_cast<float*>(addr);
      g_scratch[dev].store(ptr, std::memory_order_release);
    }
  }
  *out = ptr;
  return FHOG_OK;
}

}  // namespace

int fhog_attention_bwdbwd(fhog_stream_t stream, const void* q, const void* k, const void* v, const void* o,
                          const void* dout, const void* ddq, const void* ddk, const void* ddv, const float* lse,
                          void* dq2, void* dk2, void* dv2, void* ddo, float* delta, float* ddelta, float* bstat,
                          int batch, int n_q, int n_k, int heads, int kv_heads, int head_dim, int dtype, int causal,
                          float scale) {
  return bwdbwd_impl("fhog_attention_bwdbwd", 3, stream, q, k, v, o, dout, ddq, ddk, ddv, lse, dq2, dk2, dv2,
                     ddo, delta, ddelta, bstat, batch, n_q, n_k, heads, kv_heads, head_dim, dtype, causal, scale);
}

int fhog_attention_bwdbwd_stage(fhog_stream_t stream, int stage, const void* q, const void* k, const void* v,
                                const void* o, const void* dout, const void* ddq, const void* ddk,
                                const void* ddv, const float* lse, void* dq2, void* dk2, void* dv2, void* ddo,
                                float* delta, float* ddelta, float* bstat, int batch, int n_q, int n_k,
                                int heads, int kv_heads, int head_dim, int dtype, int causal, float scale) {
  static const char* who = "fhog_attention_bwdbwd_stage";
  if (stage != 1 && stage != 2) return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: stage must be 1 or 2, got %d", who, stage);
  return bwdbwd_impl(who, stage, stream, q, k, v, o, dout, ddq, ddk, ddv, lse, dq2, dk2, dv2, ddo, delta,
                     ddelta, bstat, batch, n_q, n_k, heads, kv_heads, head_dim, dtype, causal, scale);
}

int fhog_attention_bwdbwd_noalloc(fhog_stream_t stream, const void* q, const void* k, const void* v,
                                  const void* o, const void* dout, const void* ddq, const void* ddk,
                                  const void* ddv, const float* lse, void* dq2, void* dk2, void* dv2, void* ddo,
                                  int batch, int n_q, int n_k, int heads, int kv_heads, int head_dim, int dtype,
                                  int causal, float scale) {
  static const char* who = "fhog_attention_bwdbwd_noalloc";
  const Shape s{batch, n_q, n_k, heads, kv_heads, head_dim, dtype, causal, scale};
  if (int st = check_shape(s, who)) return st;
  if (int st = check_ptrs(who, {{"q", q}, {"k", k}, {"v", v}, {"o", o}, {"dout", dout}, {"ddq", ddq},
                                {"ddk", ddk}, {"ddv", ddv}, {"dq2", dq2}, {"dk2", dk2}, {"dv2", dv2},
                                {"ddo", ddo}},
                           {{"lse", lse}}))
    return st;
  const long long rows = (long long)batch * heads * n_q;
  if (rows > kScratchRows)
    return fail(FHOG_ERR_UNSUPPORTED,
                "%s: batch * heads * n_q = %lld exceeds the static scratch's %lld rows; use fhog_attention_bwdbwd "
                "with caller-owned row statistics",
                who, rows, kScratchRows);
  float* ws = nullptr;
  if (int st = scratch_address(who, (hipStream_t)stream, &ws)) return st;
  return bwdbwd_impl(who, 3, stream, q, k, v, o, dout, ddq, ddk, ddv, lse, dq2, dk2, dv2, ddo, ws,
                     ws + kScratchRows, ws + 2 * kScratchRows, batch, n_q, n_k, heads, kv_heads, head_dim, dtype,
                     causal, scale);
}

size_t fhog_window_workspace_bytes(int batch, int n_q, int n_k, int heads, int kv_heads, int head_dim, int dtype,
                                   int causal, int window, int sinks) {
  const Shape s{batch, n_q, n_k, heads, kv_heads, head_dim, dtype, causal, 1.0f};
  Window w;
  if (check_window(s, window, sinks, &w, "fhog_window_workspace_bytes")) return 0;
  return sink_parts_bytes(s, w);
}

int fhog_window_attention_fwd(fhog_stream_t stream, const void* q, const void* k, const void* v, void* o, float* lse,
                              int batch, int n_q, int n_k, int heads, int kv_heads, int head_dim, int dtype,
                              int causal, int window, int sinks, float scale) {
  static const char* who = "fhog_window_attention_fwd";
  const Shape s{batch, n_q, n_k, heads, kv_heads, head_dim, dtype, causal, scale};
  Window w;
  if (int st = check_window(s, window, sinks, &w, who)) return st;
  if (int st = check_ptrs(who, {{"q", q}, {"k", k}, {"v", v}, {"o", o}}, {{"lse", lse}})) return st;
  auto run = [&]<typename T, int D>() {
    fhog::FwdParams<T> p{(const T*)q, (const T*)k, (const T*)v, (T*)o,    lse,   batch,    n_q,
                         n_k,         heads,       kv_heads,    s.coff(), scale, w.window, w.sinks};
    return fhog::launch_fwd<T, D, fhog::kWindow>(p, (hipStream_t)stream);
  };
  return launch_status(dispatch(dtype, head_dim, run), who);
}

int fhog_window_attention_bwd(fhog_stream_t stream, const void* q, const void* k, const void* v, const void* o,
                              const void* dout, const float* lse, void* dq, void* dk, void* dv, float* delta,
                              void* workspace, int batch, int n_q, int n_k, int heads, int kv_heads, int head_dim,
                              int dtype, int causal, int window, int sinks, float scale) {
  static const char* who = "fhog_window_attention_bwd";
  const Shape s{batch, n_q, n_k, heads, kv_heads, head_dim, dtype, causal, scale};
  Window w;
  if (int st = check_window(s, window, sinks, &w, who)) return st;
  if (int st = check_ptrs(who, {{"q", q}, {"k", k}, {"v", v}, {"o", o}, {"dout", dout}, {"dq", dq}, {"dk", dk},
                                {"dv", dv}},
                           {{"lse", lse}, {"delta", delta}}))
    return st;
  if (int st = check_workspace(who, w, workspace)) return st;
  auto run = [&]<typename T, int D>() {
    fhog::BwdParams<T> p{(const T*)q, (const T*)k, (const T*)v, (const T*)o, (const T*)dout, lse,
                         (T*)dq, (T*)dk, (T*)dv, delta, batch, n_q, n_k, heads, kv_heads, s.coff(), scale,
                         w.window, w.sinks, w.sink, (float*)workspace};
    return fhog::launch_window_bwd<T, D>(p, (hipStream_t)stream);
  };
  return launch_status(dispatch(dtype, head_dim, run), who);
}

int fhog_window_attention_bwdbwd(fhog_stream_t stream, const void* q, const void* k, const void* v, const void* o,
                                 const void* dout, const void* ddq, const void* ddk, const void* ddv,
                                 const float* lse, void* dq2, void* dk2, void* dv2, void* ddo, float* delta,
                                 float* ddelta, float* bstat, void* workspace, int batch, int n_q, int n_k, int heads,
                                 int kv_heads, int head_dim, int dtype, int causal, int window, int sinks,
                                 float scale) {
  static const char* who = "fhog_window_attention_bwdbwd";
  const Shape s{batch, n_q, n_k, heads, kv_heads, head_dim, dtype, causal, scale};
  Window w;
  if (int st = check_window(s, window, sinks, &w, who)) return st;
  if (int st = check_ptrs(who, {{"q", q}, {"k", k}, {"v", v}, {"o", o}, {"dout", dout}, {"ddq", ddq}, {"ddk", ddk},
                                {"ddv", ddv}, {"dq2", dq2}, {"dk2", dk2}, {"dv2", dv2}, {"ddo", ddo}},
                           {{"lse", lse}, {"delta", delta}, {"ddelta", ddelta}, {"bstat", bstat}}))
    return st;
  if (int st = check_workspace(who, w, workspace)) return st;
  auto run = [&]<typename T, int D>() {
    fhog::BwdBwdParams<T> p{(const T*)q,   (const T*)k,   (const T*)v,   (const T*)o, (const T*)dout,
                            (const T*)ddq, (const T*)ddk, (const T*)ddv, lse,         (T*)dq2,
                            (T*)dk2,       (T*)dv2,       (T*)ddo,       delta,       ddelta,
                            bstat,         batch,         n_q,           n_k,         heads,
                            kv_heads,      s.coff(),      scale,         w.window,    w.sinks,
                            w.sink,        (float*)workspace};
    return fhog::launch_window_bwdbwd<T, D>(p, (hipStream_t)stream);
  };
  return launch_status(dispatch(dtype, head_dim, run), who);
}

size_t fhog_paged_workspace_bytes(int batch, int total, int single, int heads, int kv_heads, int head_dim,
                                  int page_size, int pages_per_seq, int window, int sinks) {
  const Paged s{batch, total, heads, kv_heads, head_dim, 1, page_size, pages_per_seq, FHOG_DTYPE_BF16, FHOG_DTYPE_BF16};
  if (check_paged(s, "fhog_paged_workspace_bytes") || window < 0 || sinks < 0 || batch < 1 || total < 1) return 0;
  const fhog::PagedPlan plan = fhog::paged_plan(batch, total, single != 0, heads, kv_heads,
                                                head_dim, (long)page_size * pages_per_seq, window, sinks, compute_units());
  return (size_t)plan.parts * (head_dim + 2) * sizeof(float);
}

int fhog_paged_attention(fhog_stream_t stream, const void* q, const void* k_cache, const void* v_cache,
                         const void* k_scale, const void* v_scale, const int* page_table, const int* lengths,
                         const int* query_offsets, void* out, void* workspace, size_t workspace_bytes, int batch,
                         int total, int heads, int kv_heads, int head_dim, int num_pages, int page_size,
                         int pages_per_seq, int dtype, int cache_dtype, int window, int sinks, int clear_rest,
                         float scale) {
  static const char* who = "fhog_paged_attention";
  const Paged s{batch, total, heads, kv_heads, head_dim, num_pages, page_size, pages_per_seq, dtype, cache_dtype};
  if (int st = check_paged(s, who)) return st;
  if (!(scale == scale) || scale - scale != 0.0f)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: scale must be finite", who);
  if (scale == 0.0f) return fail(FHOG_ERR_UNSUPPORTED, "%s: scale must be nonzero", who);
  if (window < 0 || sinks < 0 || (sinks > 0 && window == 0))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: window must be >= 1 (or 0: none) and sinks >= 0 (0 without a window)", who);
  if (query_offsets == nullptr && total != batch)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: without query_offsets there is one row a sequence: %d rows, %d sequences",
                who, total, batch);
  if (total == 0) return ok();
  if (batch == 0) return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: rows without a sequence", who);
  if (int st = check_ptrs(who, {{"q", q}, {"out", out}}, {})) return st;
  if (int st = check_cache(who, s, k_cache, v_cache, k_scale, v_scale, page_table, lengths)) return st;
  if (query_offsets != nullptr && !aligned(query_offsets, 4))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: query_offsets is not 4-byte aligned", who);
  const int most = 1 << 30;  // (positions are below it)
  if (window > most) window = most;
  if (sinks > most) sinks = most;
  const fhog::PagedPlan plan = fhog::paged_plan(batch, total, query_offsets == nullptr, heads, kv_heads,
                                                head_dim, (long)page_size * pages_per_seq, window, sinks, compute_units());
  if ((long long)plan.slots * kv_heads >= (1ll << 23) || plan.splits > 65535)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: problem too large", who);
  const size_t need = (size_t)plan.parts * (head_dim + 2) * sizeof(float);
  if (need > 0 && (!aligned(workspace, 16) || workspace_bytes < need))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: workspace is null, not 16-byte aligned or below its %zu bytes", who, need);
  auto run = [&]<typename T, typename C, int D>() {
    fhog::PagedParams<T, C> p{(const T*)q, (T*)out,
                              {(const C*)k_cache, (const C*)v_cache, (const uint8_t*)k_scale, (const uint8_t*)v_scale},
                              cache_shape(s, page_table, lengths, query_offsets), (float*)workspace, heads, window,
                              sinks, plan.slots, plan.splits, plan.split_tiles, plan.longest_first, clear_rest, scale};
    return fhog::launch_paged_attention<T, C, D>(p, plan.rows, (hipStream_t)stream);
  };
  return launch_status(dispatch_paged(s, run), who);
}

int fhog_paged_cache_write(fhog_stream_t stream, const void* k, const void* v, void* k_cache, void* v_cache,
                           void* k_scale, void* v_scale, const int* page_table, const int* lengths,
                           const int* query_offsets, int batch, int total, int kv_heads, int head_dim, int num_pages,
                           int page_size, int pages_per_seq, int dtype, int cache_dtype) {
  static const char* who = "fhog_paged_cache_write";
  const Paged s{batch, total, kv_heads, kv_heads, head_dim, num_pages, page_size, pages_per_seq, dtype, cache_dtype};
  if (int st = check_paged(s, who)) return st;
  if (query_offsets == nullptr && total != batch)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: without query_offsets there is one row a sequence: %d rows, %d sequences",
                who, total, batch);
  if (total == 0 || batch == 0) return ok();
  if (int st = check_ptrs(who, {{"k", k}, {"v", v}}, {})) return st;
  if (int st = check_cache(who, s, k_cache, v_cache, k_scale, v_scale, page_table, lengths)) return st;
  if (query_offsets != nullptr && !aligned(query_offsets, 4))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: query_offsets is not 4-byte aligned", who);
  auto run = [&]<typename T, typename C, int D>() {
    fhog::CacheWriteParams<T, C> p{(const T*)k, (const T*)v, (C*)k_cache, (C*)v_cache, (uint8_t*)k_scale,
                                   (uint8_t*)v_scale, cache_shape(s, page_table, lengths, query_offsets)};
    return fhog::launch_cache_write<T, C, D>(p, (hipStream_t)stream);
  };
  return launch_status(dispatch_paged(s, run), who);
}

int fhog_paged_cache_read(fhog_stream_t stream, const void* k_cache, const void* v_cache, const void* k_scale,
                          const void* v_scale, const int* page_table, const int* lengths, void* k, void* v, int batch,
                          int max_length, int kv_heads, int head_dim, int num_pages, int page_size,
                          int pages_per_seq, int dtype, int cache_dtype) {
  static const char* who = "fhog_paged_cache_read";
  const Paged s{batch, 0, kv_heads, kv_heads, head_dim, num_pages, page_size, pages_per_seq, dtype, cache_dtype};
  if (int st = check_paged(s, who)) return st;
  if (max_length < 0) return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: sizes must not be negative", who);
  if ((double)batch * max_length * kv_heads * head_dim >= kMostElements)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: problem too large", who);
  if (batch == 0 || max_length == 0) return ok();
  if (int st = check_ptrs(who, {{"k", k}, {"v", v}}, {})) return st;
  if (int st = check_cache(who, s, k_cache, v_cache, k_scale, v_scale, page_table, lengths)) return st;
  auto run = [&]<typename T, typename C, int D>() {
    fhog::CacheReadParams<T, C> p{
        {(const C*)k_cache, (const C*)v_cache, (const uint8_t*)k_scale, (const uint8_t*)v_scale},
        (T*)k, (T*)v, cache_shape(s, page_table, lengths, nullptr), max_length};
    return fhog::launch_cache_read<T, C, D>(p, (hipStream_t)stream);
  };
  return launch_status(dispatch_paged(s, run), who);
}

}  // extern "C"

namespace {

int check_rotary(const char* who, const fhog_rotary* s) {
  if (s == nullptr) return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: shape is null", who);
  if (s->batch < 0 || s->tokens < 0) return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: sizes must not be negative", who);
  if (s->heads < 1 || s->kv_heads < 1)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: sizes must be >= 1 (heads=%d kv_heads=%d)", who, s->heads, s->kv_heads);
  if (s->dtype != FHOG_DTYPE_F32 && s->dtype != FHOG_DTYPE_F16 && s->dtype != FHOG_DTYPE_BF16)
    return fail(FHOG_ERR_UNSUPPORTED, "%s: dtype must be bf16, fp16 or fp32, got %d", who, s->dtype);
  if (s->weight_dtype != s->dtype && s->weight_dtype != FHOG_DTYPE_F32)
    return fail(FHOG_ERR_UNSUPPORTED, "%s: weights must be of dtype %d or fp32, got %d", who, s->dtype, s->weight_dtype);
  if (s->head_dim < 1 || s->head_dim > 256)
    return fail(FHOG_ERR_UNSUPPORTED, "%s: head_dim must be 1 to 256, got %d", who, s->head_dim);
  if (s->rotated < 0 || s->rotated > s->head_dim || s->rotated % 2 != 0)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: rotated must be even, 0 to head_dim, got %d", who, s->rotated);
  if (s->norm && !(s->eps >= 0.0f && s->eps - s->eps == 0.0f))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: eps must be finite and >= 0", who);
  if (s->rotated > 0 && !aligned(s->frequencies, 4))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: frequencies is null or not 4-byte aligned", who);
  if (s->positions != nullptr) {
    if (s->lengths != nullptr) return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: positions and lengths exclude each other", who);
    if ((s->position_bytes != 4 && s->position_bytes != 8) || !aligned(s->positions, s->position_bytes))
      return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: positions must be aligned elements of 4 or 8 bytes", who);
    if (s->position_rows != 1 && s->position_rows != s->batch)
      return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: positions must have 1 or batch rows, got %d", who, s->position_rows);
  }
  if (s->lengths != nullptr) {
    if (!aligned(s->lengths, 4) || (s->query_offsets != nullptr && !aligned(s->query_offsets, 4)))
      return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: lengths and query_offsets must be 4-byte aligned", who);
    if (s->batch != 1) return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: packed tokens have batch 1, got %d", who, s->batch);
    if (s->tokens > 0 && s->sequences < 1)
      return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: rows without a sequence", who);
    if (s->query_offsets == nullptr && s->sequences != s->tokens)
      return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: without query_offsets there is one row a sequence: %d rows, %d sequences",
                  who, s->tokens, s->sequences);
  } else if (s->query_offsets != nullptr) {
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: query_offsets needs lengths", who);
  }
  const double tokens = (double)s->batch * s->tokens;
  if (tokens >= (1ll << 40) || tokens * (s->heads > s->kv_heads ? s->heads : s->kv_heads) * s->head_dim >= kMostElements ||
      s->heads >= (1 << 24) || s->kv_heads >= (1 << 24))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: problem too large", who);
  return FHOG_OK;
}

fhog::RotaryShape rotary_shape(const fhog_rotary& s) {
  return fhog::RotaryShape{s.batch, s.tokens, {s.heads, s.kv_heads}, s.head_dim, s.rotated, s.interleaved != 0,
                           s.norm != 0, s.weight_dtype == FHOG_DTYPE_F32 && s.dtype != FHOG_DTYPE_F32, s.eps,
                           s.frequencies, s.positions, s.position_bytes, s.position_rows, s.lengths, s.query_offsets,
                           s.sequences};
}
void rotary_strides(const fhog_rotary& s, fhog::RowStrides out[2]) {
  out[0] = {(long)s.q_stride[0], (long)s.q_stride[1], (long)s.q_stride[2]};
  out[1] = {(long)s.k_stride[0], (long)s.k_stride[1], (long)s.k_stride[2]};
}
// Whether rows can be read in pieces of kRotaryPairs elements, a lane's two pieces whole pairs: `rows` are the tensors;
// strided: q and k, with their strides, are among them.
bool rotary_wide(const fhog_rotary& s, bool strided, std::initializer_list<const void*> rows) {
  constexpr int pairs = fhog::kRotaryPairs;
  const int item = s.dtype == FHOG_DTYPE_F32 ? 4 : 2, bytes = pairs * item;
  if (s.head_dim % (2 * pairs) != 0 || s.rotated % (2 * pairs) != 0) return false;
  for (const void* p : rows)
    if (p != nullptr && !aligned(p, bytes)) return false;
  for (int i = 0; strided && i < 3; ++i)
    if (s.q_stride[i] * item % bytes != 0 || s.k_stride[i] * item % bytes != 0) return false;
  return true;
}
template <typename F> hipError_t dispatch_rows(int dtype, F&& f) {
  if (dtype == FHOG_DTYPE_BF16) return f.template operator()<__bf16>();
  if (dtype == FHOG_DTYPE_F16) return f.template operator()<_Float16>();
  return f.template operator()<float>();
}
int check_rows(const char* who, const fhog_rotary& s, std::initializer_list<std::pair<const char*, const void*>> rows) {
  const uintptr_t item = s.dtype == FHOG_DTYPE_F32 ? 4 : 2;
  for (const auto& p : rows)
    if (!aligned(p.second, item))
      return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: %s is null or not aligned to its elements", who, p.first);
  return FHOG_OK;
}
// The weights, and what stands or falls with them.
int check_weights(const char* who, const fhog_rotary& s, const void* q_weight, const void* k_weight,
                  std::initializer_list<std::pair<const void*, const void*>> more) {
  const uintptr_t item = s.weight_dtype == FHOG_DTYPE_F32 ? 4 : 2;
  auto good = [&](const void* p) { return p == nullptr || aligned(p, item); };
  if (!s.norm && (q_weight != nullptr || k_weight != nullptr))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: weights need norms", who);
  if (!good(q_weight) || !good(k_weight))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: a weight is not aligned to its elements", who);
  for (const auto& p : more) {
    if ((p.first != nullptr) != (q_weight != nullptr) || (p.second != nullptr) != (k_weight != nullptr))
      return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: a weight's derivative is null where the weight is not, or the reverse", who);
    if (!good(p.first) || !good(p.second))
      return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: a weight's derivative is not aligned to its elements", who);
  }
  return FHOG_OK;
}
// Clears the weights' gradients of a call without rows.
int clear_weights(const char* who, const fhog_rotary& s, void* const out[2], hipStream_t stream) {
  return launch_status(dispatch_rows(s.dtype, [&]<typename T>() {
    return fhog::sum_rotary_weights<T>(nullptr, out, rotary_shape(s), 0, stream);
  }), who);
}

}  // namespace

extern "C" {

size_t fhog_qk_norm_rotary_workspace_bytes(const fhog_rotary* shape) {
  if (check_rotary("fhog_qk_norm_rotary_workspace_bytes", shape) || !shape->norm) return 0;
  const long tokens = (long)shape->batch * shape->tokens;
  return (size_t)2 * fhog::rotary_grid(tokens, shape->heads, shape->head_dim, compute_units()).groups * shape->head_dim * sizeof(float);
}

int fhog_qk_norm_rotary_fwd(fhog_stream_t stream, const fhog_rotary* shape, const void* q, const void* k,
                            const void* q_weight, const void* k_weight, void* q_out, void* k_out) {
  static const char* who = "fhog_qk_norm_rotary_fwd";
  if (int st = check_rotary(who, shape)) return st;
  const fhog_rotary& s = *shape;
  if (int st = check_weights(who, s, q_weight, k_weight, {})) return st;
  const long tokens = (long)s.batch * s.tokens;
  if (tokens == 0) return ok();
  if (int st = check_rows(who, s, {{"q", q}, {"k", k}, {"q_out", q_out}, {"k_out", k_out}})) return st;
  auto run = [&]<typename T>() {
    fhog::RotaryFwdParams<T> p{{(const T*)q, (const T*)k}, {q_weight, k_weight}, {(T*)q_out, (T*)k_out}, {}, rotary_shape(s)};
    rotary_strides(s, p.stride);
    return fhog::launch_rotary_fwd<T>(p, fhog::rotary_grid(tokens, s.heads, s.head_dim, compute_units()),
                                      rotary_wide(s, true, {q, k, q_out, k_out}), (hipStream_t)stream);
  };
  return launch_status(dispatch_rows(s.dtype, run), who);
}

int fhog_qk_norm_rotary_bwd(fhog_stream_t stream, const fhog_rotary* shape, const void* q, const void* k,
                            const void* q_weight, const void* k_weight, const void* dq_out, const void* dk_out,
                            void* dq, void* dk, void* dq_weight, void* dk_weight, void* workspace) {
  static const char* who = "fhog_qk_norm_rotary_bwd";
  if (int st = check_rotary(who, shape)) return st;
  const fhog_rotary& s = *shape;
  if (int st = check_weights(who, s, q_weight, k_weight, {{dq_weight, dk_weight}})) return st;
  const long tokens = (long)s.batch * s.tokens;
  void* const dw[2] = {dq_weight, dk_weight};
  if (tokens == 0) return clear_weights(who, s, dw, (hipStream_t)stream);
  if (int st = check_rows(who, s, {{"dq_out", dq_out}, {"dk_out", dk_out}, {"dq", dq}, {"dk", dk}})) return st;
  if (s.norm)
    if (int st = check_rows(who, s, {{"q", q}, {"k", k}})) return st;
  const bool parts = dq_weight != nullptr || dk_weight != nullptr;
  if (parts && !aligned(workspace, 4))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: workspace is null or not 4-byte aligned", who);
  auto run = [&]<typename T>() {
    fhog::RotaryBwdParams<T> p{{(const T*)q, (const T*)k}, {q_weight, k_weight}, {(const T*)dq_out, (const T*)dk_out},
                               {(T*)dq, (T*)dk}, parts ? (float*)workspace : nullptr, {dq_weight, dk_weight}, {},
                               rotary_shape(s)};
    rotary_strides(s, p.stride);
    const bool wide = rotary_wide(s, s.norm, {s.norm ? q : nullptr, s.norm ? k : nullptr, dq_out, dk_out, dq, dk});
    return fhog::launch_rotary_bwd<T>(p, fhog::rotary_grid(tokens, s.heads, s.head_dim, compute_units()), wide, (hipStream_t)stream);
  };
  return launch_status(dispatch_rows(s.dtype, run), who);
}

int fhog_qk_norm_rotary_bwdbwd(fhog_stream_t stream, const fhog_rotary* shape, const void* q, const void* k,
                               const void* q_weight, const void* k_weight, const void* dq_out, const void* dk_out,
                               const void* ddq, const void* ddk, const void* ddq_weight, const void* ddk_weight,
                               void* dq2, void* dk2, void* dq_weight2, void* dk_weight2, void* ddq_out, void* ddk_out,
                               void* workspace) {
  static const char* who = "fhog_qk_norm_rotary_bwdbwd";
  if (int st = check_rotary(who, shape)) return st;
  const fhog_rotary& s = *shape;
  if (!s.norm) return fail(FHOG_ERR_UNSUPPORTED, "%s: without norms the backward is linear", who);
  if (int st = check_weights(who, s, q_weight, k_weight, {{ddq_weight, ddk_weight}, {dq_weight2, dk_weight2}})) return st;
  const long tokens = (long)s.batch * s.tokens;
  void* const dw[2] = {dq_weight2, dk_weight2};
  if (tokens == 0) return clear_weights(who, s, dw, (hipStream_t)stream);
  if (int st = check_rows(who, s, {{"q", q}, {"k", k}, {"dq_out", dq_out}, {"dk_out", dk_out}, {"ddq", ddq}, {"ddk", ddk},
                                   {"dq2", dq2}, {"dk2", dk2}, {"ddq_out", ddq_out}, {"ddk_out", ddk_out}}))
    return st;
  const bool parts = dq_weight2 != nullptr || dk_weight2 != nullptr;
  if (parts && !aligned(workspace, 4))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: workspace is null or not 4-byte aligned", who);
  auto run = [&]<typename T>() {
    fhog::RotaryBwdBwdParams<T> p{{(const T*)q, (const T*)k}, {q_weight, k_weight},
                                  {(const T*)dq_out, (const T*)dk_out}, {(const T*)ddq, (const T*)ddk},
                                  {ddq_weight, ddk_weight}, {(T*)dq2, (T*)dk2}, {(T*)ddq_out, (T*)ddk_out},
                                  parts ? (float*)workspace : nullptr, {dq_weight2, dk_weight2}, {}, rotary_shape(s)};
    rotary_strides(s, p.stride);
    const bool wide = rotary_wide(s, true, {q, k, dq_out, dk_out, ddq, ddk, dq2, dk2, ddq_out, ddk_out});
    return fhog::launch_rotary_bwdbwd<T>(p, fhog::rotary_grid(tokens, s.heads, s.head_dim, compute_units()), wide, (hipStream_t)stream);
  };
  return launch_status(dispatch_rows(s.dtype, run), who);
}

}  // extern "C"

namespace {

// What the allocator's two entry points share.
int check_pages(const char* who, int batch, int kv_heads, int head_dim, int num_pages, int page_size, int pages_per_seq,
                int cache_dtype) {
  const int dtype = cache_dtype == FHOG_DTYPE_E4M3 ? (int)FHOG_DTYPE_BF16 : cache_dtype;
  if (int st = check_paged({batch, 0, kv_heads, kv_heads, head_dim, num_pages, page_size, pages_per_seq, dtype,
                            cache_dtype}, who))
    return st;
  if ((long long)batch * pages_per_seq >= (1ll << 31) || kv_heads > 65535)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: problem too large", who);
  return FHOG_OK;
}

int check_pages_workspace(const char* who, const void* workspace, size_t bytes, int batch, int num_pages,
                          int pages_per_seq) {
  const size_t need = fhog_paged_pages_workspace_bytes(batch, num_pages, pages_per_seq);
  if (!aligned(workspace, 4) || bytes < need)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: workspace is null, not 4-byte aligned or below its %zu bytes", who, need);
  return FHOG_OK;
}

fhog::PageBytes page_bytes(const void* k, const void* v, const void* ks, const void* vs, const void* means, int head_dim,
                           int page_size, int cache_dtype) {
  const bool quantised = cache_dtype == FHOG_DTYPE_E4M3;
  const int token = head_dim * (quantised ? 1 : 2);
  const long row = (long)token * page_size;
  return fhog::PageBytes{{(char*)k, (char*)v, quantised ? (char*)ks : nullptr, quantised ? (char*)vs : nullptr,
                          (char*)means},
                         {row, row, page_size, page_size, head_dim * 4}, {token, token, 1, 1, 0}};
}

}  // namespace

extern "C" {

size_t fhog_paged_pages_workspace_bytes(int batch, int num_pages, int pages_per_seq) {
  if (batch < 0 || num_pages < 1 || pages_per_seq < 1) return 0;
  return (size_t)fhog::pages_workspace_ints(batch, pages_per_seq, num_pages) * sizeof(int);
}

int fhog_paged_cache_extend(fhog_stream_t stream, void* k_cache, void* v_cache, void* k_scale, void* v_scale,
                            int* page_table, int* lengths, const int* parents, const int* new_tokens, int new_each,
                            int* free_pages, void* workspace, size_t workspace_bytes, int batch, int kv_heads,
                            int head_dim, int num_pages, int page_size, int pages_per_seq, int cache_dtype) {
  static const char* who = "fhog_paged_cache_extend";
  if (int st = check_pages(who, batch, kv_heads, head_dim, num_pages, page_size, pages_per_seq, cache_dtype)) return st;
  if (batch == 0) return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: no rows", who);
  if (new_tokens == nullptr && new_each < 0)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: new_each must be >= 0, got %d", who, new_each);
  const Paged s{batch, 0, kv_heads, kv_heads, head_dim, num_pages, page_size, pages_per_seq, FHOG_DTYPE_BF16, cache_dtype};
  if (int st = check_cache(who, s, k_cache, v_cache, k_scale, v_scale, page_table, lengths)) return st;
  if (int st = check_ptrs(who, {}, {{"free_pages", free_pages}})) return st;
  if ((parents != nullptr && !aligned(parents, 4)) || (new_tokens != nullptr && !aligned(new_tokens, 4)))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: parents and new_tokens must be 4-byte aligned", who);
  if (int st = check_pages_workspace(who, workspace, workspace_bytes, batch, num_pages, pages_per_seq)) return st;
  fhog::PagesParams p{page_table, lengths, parents, new_tokens, new_each, batch, pages_per_seq, num_pages,
                      __builtin_ctz((unsigned)page_size), kv_heads, 0};
  fhog::pages_workspace(p, (int*)workspace);
  return launch_status(fhog::launch_pages_extend(
      p, page_bytes(k_cache, v_cache, k_scale, v_scale, nullptr, head_dim, page_size, cache_dtype), free_pages,
      (hipStream_t)stream), who);
}

int fhog_paged_cache_compact(fhog_stream_t stream, const void* k_cache, const void* v_cache, const void* k_scale,
                             const void* v_scale, const float* key_means, const int* page_table, const int* lengths,
                             void* k_out, void* v_out, void* k_scale_out, void* v_scale_out, float* means_out,
                             int* table_out, void* workspace, size_t workspace_bytes, int batch, int kv_heads,
                             int head_dim, int num_pages, int page_size, int pages_per_seq, int out_pages,
                             int cache_dtype) {
  static const char* who = "fhog_paged_cache_compact";
  if (int st = check_pages(who, batch, kv_heads, head_dim, num_pages, page_size, pages_per_seq, cache_dtype)) return st;
  if (out_pages < 1) return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: out_pages must be >= 1, got %d", who, out_pages);
  const Paged s{batch, 0, kv_heads, kv_heads, head_dim, num_pages, page_size, pages_per_seq, FHOG_DTYPE_BF16, cache_dtype};
  if (int st = check_ptrs(who, {{"k_cache", k_cache}, {"v_cache", v_cache}, {"k_out", k_out}, {"v_out", v_out}}, {}))
    return st;
  if (batch > 0)
    if (int st = check_ptrs(who, {}, {{"page_table", page_table}, {"lengths", lengths}, {"table_out", table_out}})) return st;
  if (cache_dtype == FHOG_DTYPE_E4M3)
    if (int st = check_ptrs(who, {{"k_scale", k_scale}, {"v_scale", v_scale}, {"k_scale_out", k_scale_out},
                                  {"v_scale_out", v_scale_out}}, {}))
      return st;
  if ((key_means != nullptr) != (means_out != nullptr))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: key_means and means_out go together", who);
  if (key_means != nullptr)
    if (int st = check_ptrs(who, {{"key_means", key_means}, {"means_out", means_out}}, {})) return st;
  if (int st = check_pages_workspace(who, workspace, workspace_bytes, batch, num_pages, pages_per_seq)) return st;
  fhog::PagesParams p{const_cast<int*>(page_table), const_cast<int*>(lengths), nullptr, nullptr, 0, batch, pages_per_seq,
                      num_pages, __builtin_ctz((unsigned)page_size), kv_heads, 1};
  fhog::pages_workspace(p, (int*)workspace);
  return launch_status(fhog::launch_pages_compact(
      p, page_bytes(k_cache, v_cache, k_scale, v_scale, key_means, head_dim, page_size, cache_dtype),
      page_bytes(k_out, v_out, k_scale_out, v_scale_out, means_out, head_dim, page_size, cache_dtype), out_pages,
      table_out, (hipStream_t)stream), who);
}

}  // extern "C"

namespace {

// What tokens over chosen blocks share: the cache's sizes, and the offsets.
int check_tokens(const char* who, const Paged& s, const int* query_offsets) {
  if (query_offsets == nullptr && s.rows != s.batch)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: without query_offsets there is one row a sequence: %d rows, %d sequences",
                who, s.rows, s.batch);
  if (query_offsets != nullptr && !aligned(query_offsets, 4))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: query_offsets is not 4-byte aligned", who);
  return FHOG_OK;
}
int check_blocks(const char* who, const Paged& s, int blocks) {
  if (blocks < 1) return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: blocks must be >= 1, got %d", who, blocks);
  // (a split's blocks are listed in LDS, and a join's splits)
  if (blocks > 32768 || (long long)blocks * s.page_size > (1ll << 30))
    return fail(FHOG_ERR_UNSUPPORTED, "%s: blocks must be <= 32768 and hold at most 2^30 keys, got %d", who, blocks);
  return FHOG_OK;
}
template <typename F> hipError_t dispatch_dim(int head_dim, F&& f) {
  if (head_dim == 64) return f.template operator()<64>();
  if (head_dim == 128) return f.template operator()<128>();
  return f.template operator()<256>();
}

}  // namespace

extern "C" {

int fhog_paged_key_means(fhog_stream_t stream, const void* k_cache, const void* k_scale, float* key_means,
                         const int* page_table, const int* lengths, const int* query_offsets, int batch, int kv_heads,
                         int head_dim, int num_pages, int page_size, int pages_per_seq, int cache_dtype) {
  static const char* who = "fhog_paged_key_means";
  const int dtype = cache_dtype == FHOG_DTYPE_E4M3 ? (int)FHOG_DTYPE_BF16 : cache_dtype;
  const Paged s{batch, 0, kv_heads, kv_heads, head_dim, num_pages, page_size, pages_per_seq, dtype, cache_dtype};
  if (int st = check_paged(s, who)) return st;
  if (query_offsets != nullptr && !aligned(query_offsets, 4))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: query_offsets is not 4-byte aligned", who);
  if (batch == 0) return ok();
  if (int st = check_cache(who, s, k_cache, k_cache, k_scale, k_scale, page_table, lengths)) return st;
  if (int st = check_ptrs(who, {}, {{"key_means", key_means}})) return st;
  // How many pages the tokens fill only the device knows; single tokens fill one each at most.
  const long long most = (long long)batch * (query_offsets != nullptr ? pages_per_seq : 1) * kv_heads;
  const long long fill = 8ll * (compute_units() > 0 ? compute_units() : 256);
  const int workgroups = (int)(most < fill ? most : fill);
  fhog::CacheShape at = cache_shape(s, page_table, lengths, query_offsets);
  at.total = 0x7fffffff;
  auto run = [&]<typename C>() {
    return dispatch_dim(head_dim, [&]<int D>() {
      return fhog::launch_key_means<C, D>({(const C*)k_cache, (const uint8_t*)k_scale, key_means, at}, workgroups,
                                          (hipStream_t)stream);
    });
  };
  return launch_status(cache_dtype == FHOG_DTYPE_E4M3  ? run.template operator()<fhog::e4m3>()
                       : cache_dtype == FHOG_DTYPE_F16 ? run.template operator()<_Float16>()
                                                       : run.template operator()<__bf16>(),
                       who);
}

size_t fhog_paged_block_select_workspace_bytes(int batch, int total, int single, int kv_heads, int head_dim,
                                               int pages_per_seq, int first, int last) {
  if (batch < 1 || total < 1 || kv_heads < 1 || pages_per_seq < 1 || first < 0 || last < 1) return 0;
  return (size_t)fhog::select_plan(batch, total, single != 0, kv_heads, head_dim, pages_per_seq, first, last).slab * kv_heads *
         pages_per_seq * 8;
}

int fhog_paged_block_select(fhog_stream_t stream, const void* q, const float* key_means, const int* page_table,
                            const int* lengths, const int* query_offsets, int* chosen, void* workspace,
                            size_t workspace_bytes, int batch, int total, int heads, int kv_heads, int head_dim,
                            int num_pages, int page_size, int pages_per_seq, int dtype, int blocks, int first, int last) {
  static const char* who = "fhog_paged_block_select";
  const Paged s{batch, total, heads, kv_heads, head_dim, num_pages, page_size, pages_per_seq, dtype, dtype};
  if (int st = check_paged(s, who)) return st;
  if (int st = check_tokens(who, s, query_offsets)) return st;
  if (int st = check_blocks(who, s, blocks)) return st;
  if (first < 0 || last < 1 || (long long)first + last > blocks)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: needs first >= 0, last >= 1 and first + last <= blocks, got %d, %d and %d",
                who, first, last, blocks);
  if (total == 0) return ok();
  if (batch == 0) return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: rows without a sequence", who);
  if (pages_per_seq > (1 << 21) || kv_heads > (1 << 16) || (double)total * kv_heads * blocks >= kMostElements)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: problem too large", who);
  if (int st = check_ptrs(who, {{"q", q}, {"key_means", key_means}},
                          {{"page_table", page_table}, {"lengths", lengths}, {"chosen", chosen}}))
    return st;
  const fhog::SelectPlan plan = fhog::select_plan(batch, total, query_offsets == nullptr, kv_heads, head_dim, pages_per_seq, first, last);
  if ((long long)plan.slots * kv_heads >= (1ll << 23))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: problem too large", who);
  const size_t need = fhog_paged_block_select_workspace_bytes(batch, total, query_offsets == nullptr, kv_heads, head_dim,
                                                              pages_per_seq, first, last);
  if (need > 0 && (!aligned(workspace, 8) || workspace_bytes < need))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: workspace is null, not 8-byte aligned or below its %zu bytes", who, need);
  auto run = [&]<typename T>() {
    return dispatch_dim(head_dim, [&]<int D>() {
      fhog::BlockSelectParams<T> p{(const T*)q, key_means, chosen, cache_shape(s, page_table, lengths, query_offsets),
                                   (unsigned long*)workspace, heads, blocks, first, last};
      return fhog::launch_block_select<T, D>(p, plan, (hipStream_t)stream);
    });
  };
  return launch_status(dtype == FHOG_DTYPE_BF16 ? run.template operator()<__bf16>() : run.template operator()<_Float16>(),
                       who);
}

size_t fhog_paged_block_workspace_bytes(int batch, int total, int single, int heads, int kv_heads, int head_dim,
                                        int page_size, int pages_per_seq, int blocks) {
  static const char* who = "fhog_paged_block_workspace_bytes";
  const Paged s{batch, total, heads, kv_heads, head_dim, 1, page_size, pages_per_seq, FHOG_DTYPE_BF16, FHOG_DTYPE_BF16};
  if (check_paged(s, who) || check_blocks(who, s, blocks) || batch < 1 || total < 1) return 0;
  if (fhog::block_chunk_rule(batch, total, heads, kv_heads, head_dim, page_size, pages_per_seq, blocks, single != 0))
    return fhog::block_chunk_plan(batch, total, heads, kv_heads, head_dim, pages_per_seq, blocks).bytes;
  const fhog::BlockPlan plan = fhog::block_plan(total, heads, kv_heads, head_dim, page_size, blocks, compute_units());
  return (size_t)plan.parts * (head_dim + 2) * sizeof(float);
}

int fhog_paged_block_attention(fhog_stream_t stream, const void* q, const int* chosen, const void* k_cache,
                               const void* v_cache, const void* k_scale, const void* v_scale, const int* page_table,
                               const int* lengths, const int* query_offsets, void* out, void* workspace,
                               size_t workspace_bytes, int batch, int total, int heads, int kv_heads, int head_dim,
                               int num_pages, int page_size, int pages_per_seq, int dtype, int cache_dtype, int blocks,
                               int clear_rest, float scale) {
  static const char* who = "fhog_paged_block_attention";
  const Paged s{batch, total, heads, kv_heads, head_dim, num_pages, page_size, pages_per_seq, dtype, cache_dtype};
  if (int st = check_paged(s, who)) return st;
  if (!(scale == scale) || scale - scale != 0.0f)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: scale must be finite", who);
  if (scale == 0.0f) return fail(FHOG_ERR_UNSUPPORTED, "%s: scale must be nonzero", who);
  if (int st = check_tokens(who, s, query_offsets)) return st;
  if (int st = check_blocks(who, s, blocks)) return st;
  if (total == 0) return ok();
  if (batch == 0) return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: rows without a sequence", who);
  if (int st = check_ptrs(who, {{"q", q}, {"out", out}}, {{"chosen", chosen}})) return st;
  if (int st = check_cache(who, s, k_cache, v_cache, k_scale, v_scale, page_table, lengths)) return st;
  const long long tiles = (long long)total * ((heads / kv_heads + 15) / 16);
  if (tiles * kv_heads >= (1ll << 23) || (double)total * kv_heads * blocks >= kMostElements)
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: problem too large", who);
  const size_t need = fhog_paged_block_workspace_bytes(batch, total, query_offsets == nullptr, heads, kv_heads, head_dim,
                                                       page_size, pages_per_seq, blocks);
  if (need > 0 && (!aligned(workspace, 16) || workspace_bytes < need))
    return fail(FHOG_ERR_INVALID_ARGUMENT, "%s: workspace is null, not 16-byte aligned or below its %zu bytes", who, need);
  if (fhog::block_chunk_rule(batch, total, heads, kv_heads, head_dim, page_size, pages_per_seq, blocks, query_offsets == nullptr)) {
    const fhog::BlockChunkPlan plan = fhog::block_chunk_plan(batch, total, heads, kv_heads, head_dim, pages_per_seq, blocks);
    auto run = [&]<typename T, typename C, int D>() {
      fhog::BlockChunkParams<T, C> p{(const T*)q, (T*)out,
                                     {(const C*)k_cache, (const C*)v_cache, (const uint8_t*)k_scale, (const uint8_t*)v_scale},
                                     cache_shape(s, page_table, lengths, query_offsets), chosen, heads, blocks, clear_rest,
                                     scale, (int)plan.lists};
      fhog::block_chunk_workspace(p, plan, D, workspace);
      return fhog::launch_block_chunk<T, C, D>(p, plan.slab, (hipStream_t)stream);
    };
    return launch_status(dispatch_paged(s, run), who);
  }
  const fhog::BlockPlan plan = fhog::block_plan(total, heads, kv_heads, head_dim, page_size, blocks, compute_units());
  auto run = [&]<typename T, typename C, int D>() {
    fhog::BlockParams<T, C> p{(const T*)q, (T*)out,
                              {(const C*)k_cache, (const C*)v_cache, (const uint8_t*)k_scale, (const uint8_t*)v_scale},
                              cache_shape(s, page_table, lengths, query_offsets), chosen, (float*)workspace, heads, blocks,
                              plan.slots, plan.splits, plan.split_tiles, clear_rest, scale, 0};
    return fhog::launch_block_attention<T, C, D>(p, plan.slab, (hipStream_t)stream);
  };
  return launch_status(dispatch_paged(s, run), who);
}

}  // extern "C"
