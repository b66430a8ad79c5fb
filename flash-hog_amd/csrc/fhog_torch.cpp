// Tensor-level front door to the C ABI for eager callers, as a torch C++
// extension (flash_hog/_lib/_fhog_torch*.so, built by flash-hog_amd/build.py).
//
// It does in C++ what flash_hog/_hip.py's attention_fwd / attention_bwd /
// attention_bwdbwd do in Python (the same checks with the same messages, the
// same allocations, the caller's device made current around the call, the
// current stream of that device) and then calls the C-ABI entry point, so a
// call costs a few microseconds of host time instead of the Python wrapper's
// 9-20 us. That host time is what bounds an eager Hessian-vector product at
// short sequences, whose GPU work is shorter than the host's.
//
// The entry points are not linked: bind() receives their addresses from the
// library _hip.py loaded (which honours its FLASH_HOG_HIP_LIB override), and
// the Python exception class to raise for a non-zero status. _hip.py uses this
// module when it is built and falls back to its own wrappers when it is not;
// both reach the same kernels.
//
// attention() is dot_product_attention's eager autograd path in C++: two
// torch::autograd::Function nodes with the rules of
// flash_hog/torch/attention.py (the forward saving (q, k, v, L, O); its
// backward, itself differentiable once, saving (q, k, v, O, L, dO); the double
// backward with no cotangent for L and O), so that a Hessian-vector product
// runs no Python between the autograd engine and the kernels.
//
// The calls themselves (the *_core functions) touch no Python object: the
// autograd engine runs backward nodes on its own threads, without the GIL.
// They throw ArgError and StatusError; the Python-facing functions release the
// GIL around them and turn those into ValueError and the bound FlashHogError.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include <cstdint>
#include <sstream>
#include <algorithm>
#include <stdexcept>
#include <string>
#include <tuple>

#include "flash_hog.h"

namespace py = pybind11;

namespace {

struct Api {
  decltype(&fhog_attention_fwd) fwd = nullptr;
  decltype(&fhog_attention_bwd) bwd = nullptr;
  decltype(&fhog_attention_bwdbwd) bwdbwd = nullptr;
  decltype(&fhog_last_error) last_error = nullptr;
  decltype(&fhog_status_string) status_string = nullptr;
  decltype(&fhog_window_workspace_bytes) window_bytes = nullptr;
  decltype(&fhog_window_attention_fwd) window_fwd = nullptr;
  decltype(&fhog_window_attention_bwd) window_bwd = nullptr;
  decltype(&fhog_window_attention_bwdbwd) window_bwdbwd = nullptr;
  decltype(&fhog_paged_workspace_bytes) paged_bytes = nullptr;
  decltype(&fhog_paged_attention) paged_attention = nullptr;
  decltype(&fhog_paged_cache_write) cache_write = nullptr;
  decltype(&fhog_paged_cache_read) cache_read = nullptr;
  decltype(&fhog_paged_pages_workspace_bytes) pages_bytes = nullptr;
  decltype(&fhog_paged_cache_extend) cache_extend = nullptr;
  decltype(&fhog_paged_cache_compact) cache_compact = nullptr;
  decltype(&fhog_paged_key_means) key_means = nullptr;
  decltype(&fhog_paged_block_select_workspace_bytes) select_bytes = nullptr;
  decltype(&fhog_paged_block_select) block_select = nullptr;
  decltype(&fhog_paged_block_workspace_bytes) block_bytes = nullptr;
  decltype(&fhog_paged_block_attention) block_attention = nullptr;
  decltype(&fhog_qk_norm_rotary_workspace_bytes) rotary_bytes = nullptr;
  decltype(&fhog_qk_norm_rotary_fwd) rotary_fwd = nullptr;
  decltype(&fhog_qk_norm_rotary_bwd) rotary_bwd = nullptr;
  decltype(&fhog_qk_norm_rotary_bwdbwd) rotary_bwdbwd = nullptr;
  py::object error_cls;
};

Api& api() {
  static Api a;
  return a;
}

void bind(std::uintptr_t fwd, std::uintptr_t bwd, std::uintptr_t bwdbwd, std::uintptr_t last_error,
          std::uintptr_t status_string, py::object error_cls) {
  Api& a = api();
  a.fwd = reinterpret_cast<decltype(a.fwd)>(fwd);
  a.bwd = reinterpret_cast<decltype(a.bwd)>(bwd);
  a.bwdbwd = reinterpret_cast<decltype(a.bwdbwd)>(bwdbwd);
  a.last_error = reinterpret_cast<decltype(a.last_error)>(last_error);
  a.status_string = reinterpret_cast<decltype(a.status_string)>(status_string);
  a.error_cls = std::move(error_cls);
}

void bind_window(std::uintptr_t bytes, std::uintptr_t fwd, std::uintptr_t bwd, std::uintptr_t bwdbwd) {
  Api& a = api();
  a.window_bytes = reinterpret_cast<decltype(a.window_bytes)>(bytes);
  a.window_fwd = reinterpret_cast<decltype(a.window_fwd)>(fwd);
  a.window_bwd = reinterpret_cast<decltype(a.window_bwd)>(bwd);
  a.window_bwdbwd = reinterpret_cast<decltype(a.window_bwdbwd)>(bwdbwd);
}

void bind_paged(std::uintptr_t bytes, std::uintptr_t attention, std::uintptr_t write, std::uintptr_t read) {
  Api& a = api();
  a.paged_bytes = reinterpret_cast<decltype(a.paged_bytes)>(bytes);
  a.paged_attention = reinterpret_cast<decltype(a.paged_attention)>(attention);
  a.cache_write = reinterpret_cast<decltype(a.cache_write)>(write);
  a.cache_read = reinterpret_cast<decltype(a.cache_read)>(read);
}

void bind_pages(std::uintptr_t bytes, std::uintptr_t extend, std::uintptr_t compact) {
  Api& a = api();
  a.pages_bytes = reinterpret_cast<decltype(a.pages_bytes)>(bytes);
  a.cache_extend = reinterpret_cast<decltype(a.cache_extend)>(extend);
  a.cache_compact = reinterpret_cast<decltype(a.cache_compact)>(compact);
}

void bind_blocks(std::uintptr_t means, std::uintptr_t select_bytes, std::uintptr_t select, std::uintptr_t bytes,
                 std::uintptr_t attention) {
  Api& a = api();
  a.key_means = reinterpret_cast<decltype(a.key_means)>(means);
  a.select_bytes = reinterpret_cast<decltype(a.select_bytes)>(select_bytes);
  a.block_select = reinterpret_cast<decltype(a.block_select)>(select);
  a.block_bytes = reinterpret_cast<decltype(a.block_bytes)>(bytes);
  a.block_attention = reinterpret_cast<decltype(a.block_attention)>(attention);
}

void bind_rotary(std::uintptr_t bytes, std::uintptr_t fwd, std::uintptr_t bwd, std::uintptr_t bwdbwd) {
  Api& a = api();
  a.rotary_bytes = reinterpret_cast<decltype(a.rotary_bytes)>(bytes);
  a.rotary_fwd = reinterpret_cast<decltype(a.rotary_fwd)>(fwd);
  a.rotary_bwd = reinterpret_cast<decltype(a.rotary_bwd)>(bwd);
  a.rotary_bwdbwd = reinterpret_cast<decltype(a.rotary_bwdbwd)>(bwdbwd);
}

std::string shape_str(const at::Tensor& t) {
  std::ostringstream os;
  os << "(";
  for (int64_t i = 0; i < t.dim(); ++i) os << (i ? ", " : "") << t.size(i);
  os << (t.dim() == 1 ? ",)" : ")");
  return os.str();
}

std::string dtype_str(at::ScalarType s) {
  switch (s) {
    case at::kFloat: return "torch.float32";
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    default: return std::string("torch.") + c10::toString(s);
  }
}

std::string device_str(const at::Tensor& t) {
  std::ostringstream os;
  os << t.device();
  return os.str();
}

// A bad argument (ValueError in Python) and a non-zero C-ABI status
// (FlashHogError(status, message) in Python).
struct ArgError : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct StatusError : std::runtime_error {
  int status;
  StatusError(int s, const std::string& msg) : std::runtime_error(msg), status(s) {}
};

[[noreturn]] void value_error(const std::string& msg) { throw ArgError(msg); }

int dtype_code(at::ScalarType s) {
  switch (s) {
    case at::kFloat: return FHOG_DTYPE_F32;
    case at::kHalf: return FHOG_DTYPE_F16;
    case at::kBFloat16: return FHOG_DTYPE_BF16;
    default: value_error("unsupported dtype " + dtype_str(s));
  }
}

// Every tensor on the first one's GPU device, with dtype `dtype` unless it is
// None (_hip.py _check_inputs).
void check_inputs(std::initializer_list<std::pair<const char*, const at::Tensor*>> named,
                  c10::optional<at::ScalarType> dtype) {
  const at::Tensor* first = nullptr;
  for (const auto& [name, t] : named) {
    if (!t->is_cuda()) value_error(std::string(name) + " must be on a GPU device, got " + device_str(*t));
    if (!first) {
      first = t;
    } else if (t->get_device() != first->get_device()) {
      value_error(std::string(name) + " is on " + device_str(*t) + ", expected " + device_str(*first));
    }
    if (dtype && t->scalar_type() != *dtype)
      value_error(std::string(name) + " has dtype " + dtype_str(t->scalar_type()) + ", expected " +
                  dtype_str(*dtype));
  }
}

struct Dims {
  int B, Tq, Tk, N, Nk, H;
};

// (B, Tq, Tk, N, Nk, H) of q (B, Tq, N, H) and k (B, Tk, Nk, H) (_hip.py _dims).
Dims dims(const at::Tensor& q, const at::Tensor& k) {
  if (q.dim() != 4 || k.dim() != 4)
    value_error("expected (B, T, N, H) tensors, got q" + shape_str(q) + " k" + shape_str(k));
  if (k.size(0) != q.size(0) || k.size(3) != q.size(3))
    value_error("q" + shape_str(q) + " and k" + shape_str(k) + " disagree on batch or head_dim");
  if (k.size(2) == 0 || q.size(2) % k.size(2) != 0) {
    std::ostringstream os;
    os << "query heads (" << q.size(2) << ") must be a multiple of key/value heads (" << k.size(2) << ")";
    value_error(os.str());
  }
  dtype_code(q.scalar_type());
  for (int64_t s : q.sizes())
    if (s > INT32_MAX) value_error("q" + shape_str(q) + " has a dimension beyond the C ABI's int range");
  if (k.size(1) > INT32_MAX) value_error("k" + shape_str(k) + " has a dimension beyond the C ABI's int range");
  return {(int)q.size(0), (int)q.size(1), (int)k.size(1), (int)q.size(2), (int)k.size(2), (int)q.size(3)};
}

void expect(const char* name, const at::Tensor& t, at::IntArrayRef shape,
            c10::optional<at::ScalarType> dtype = c10::nullopt) {
  if (t.sizes() != shape) {
    std::ostringstream os;
    os << "(";
    for (size_t i = 0; i < shape.size(); ++i) os << (i ? ", " : "") << shape[i];
    os << (shape.size() == 1 ? ",)" : ")");
    value_error(std::string(name) + " has shape " + shape_str(t) + ", expected " + os.str());
  }
  if (dtype && t.scalar_type() != *dtype)
    value_error(std::string(name) + " has dtype " + dtype_str(t.scalar_type()) + ", expected " + dtype_str(*dtype));
}

at::Tensor contig(const at::Tensor& t) { return t.is_contiguous() ? t : t.contiguous(); }

// The current stream of t's device (torch's, as _hip.py takes it).
fhog_stream_t current_stream(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// The message comes from the calling thread's fhog_last_error.
void check_status(int status) {
  if (status == FHOG_OK) return;
  const Api& a = api();
  std::string msg = a.last_error();
  if (msg.empty()) msg = a.status_string(status);
  throw StatusError(status, msg);
}

void require_bound(const void* fn) {
  if (!fn) throw std::runtime_error("_fhog_torch.bind() has not been called");
}

// A window of keys and sinks (0, 0: none), and the workspace that a backward with one needs
// (undefined where it needs none).
struct Window {
  int window = 0, sinks = 0;
  at::Tensor workspace(const at::Tensor& q, const Dims& d, int causal) const {
    const size_t size = api().window_bytes(d.B, d.Tq, d.Tk, d.N, d.Nk, d.H, dtype_code(q.scalar_type()), causal, window,
                                           sinks);
    return size ? at::empty({(int64_t)size}, q.options().dtype(at::kByte)) : at::Tensor();
  }
};
void* data_or_null(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

std::tuple<at::Tensor, at::Tensor> fwd_core(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_,
                                            int causal, double scale, Window w) {
  require_bound((const void*)api().fwd);
  check_inputs({{"q", &q_}, {"k", &k_}, {"v", &v_}}, q_.scalar_type());
  const Dims d = dims(q_, k_);
  expect("v", v_, k_.sizes());
  const at::Tensor q = contig(q_), k = contig(k_), v = contig(v_);
  at::Tensor o = at::empty_like(q);
  at::Tensor lse = at::empty({(int64_t)d.B, (int64_t)d.N, (int64_t)d.Tq}, q.options().dtype(at::kFloat));
  c10::DeviceGuard guard(q.device());
  const int dt = dtype_code(q.scalar_type());
  const int status =
      w.window ? api().window_fwd(current_stream(q), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                                  lse.data_ptr<float>(), d.B, d.Tq, d.Tk, d.N, d.Nk, d.H, dt, causal, w.window,
                                  w.sinks, (float)scale)
               : api().fwd(current_stream(q), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                           lse.data_ptr<float>(), d.B, d.Tq, d.Tk, d.N, d.Nk, d.H, dt, causal, (float)scale);
  check_status(status);
  return {o, lse};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> bwd_core(
    const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_, const at::Tensor& o_, const at::Tensor& dout_,
    const at::Tensor& lse_, int causal, double scale, Window w) {
  require_bound((const void*)api().bwd);
  check_inputs({{"q", &q_}, {"k", &k_}, {"v", &v_}, {"o", &o_}, {"dout", &dout_}}, q_.scalar_type());
  check_inputs({{"q", &q_}, {"lse", &lse_}}, c10::nullopt);
  const Dims d = dims(q_, k_);
  expect("v", v_, k_.sizes());
  expect("o", o_, q_.sizes());
  expect("dout", dout_, q_.sizes());
  expect("lse", lse_, {(int64_t)d.B, (int64_t)d.N, (int64_t)d.Tq}, at::kFloat);
  const at::Tensor q = contig(q_), k = contig(k_), v = contig(v_), o = contig(o_), dout = contig(dout_),
                   lse = contig(lse_);
  at::Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v);
  at::Tensor delta = at::empty({(int64_t)d.B, (int64_t)d.N, (int64_t)d.Tq}, q.options().dtype(at::kFloat));
  c10::DeviceGuard guard(q.device());
  const int dt = dtype_code(q.scalar_type());
  int status;
  if (w.window) {
    const at::Tensor ws = w.workspace(q, d, causal);
    status = api().window_bwd(current_stream(q), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                              dout.data_ptr(), lse.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                              delta.data_ptr<float>(), data_or_null(ws), d.B, d.Tq, d.Tk, d.N, d.Nk, d.H, dt, causal,
                              w.window, w.sinks, (float)scale);
  } else {
    status = api().bwd(current_stream(q), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), dout.data_ptr(),
                       lse.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), delta.data_ptr<float>(),
                       d.B, d.Tq, d.Tk, d.N, d.Nk, d.H, dt, causal, (float)scale);
  }
  check_status(status);
  return {dq, dk, dv, delta};
}

// dq2, dk2, dv2, ddo and the (3, B, N, Tq) fp32 row statistics D, dD, B.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> bwdbwd_core(
    const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_, const at::Tensor& o_, const at::Tensor& dout_,
    const at::Tensor& ddq_, const at::Tensor& ddk_, const at::Tensor& ddv_, const at::Tensor& lse_, int causal,
    double scale, Window w) {
  require_bound((const void*)api().bwdbwd);
  check_inputs({{"q", &q_}, {"k", &k_}, {"v", &v_}, {"o", &o_}, {"dout", &dout_}, {"ddq", &ddq_}, {"ddk", &ddk_},
                {"ddv", &ddv_}},
               q_.scalar_type());
  check_inputs({{"q", &q_}, {"lse", &lse_}}, c10::nullopt);
  const Dims d = dims(q_, k_);
  expect("v", v_, k_.sizes());
  expect("o", o_, q_.sizes());
  expect("dout", dout_, q_.sizes());
  expect("ddq", ddq_, q_.sizes());
  expect("ddk", ddk_, k_.sizes());
  expect("ddv", ddv_, k_.sizes());
  expect("lse", lse_, {(int64_t)d.B, (int64_t)d.N, (int64_t)d.Tq}, at::kFloat);
  const at::Tensor q = contig(q_), k = contig(k_), v = contig(v_), o = contig(o_), dout = contig(dout_),
                   ddq = contig(ddq_), ddk = contig(ddk_), ddv = contig(ddv_), lse = contig(lse_);
  at::Tensor dq2 = at::empty_like(q), dk2 = at::empty_like(k), dv2 = at::empty_like(v), ddo = at::empty_like(dout);
  at::Tensor stats = at::empty({3, (int64_t)d.B, (int64_t)d.N, (int64_t)d.Tq}, q.options().dtype(at::kFloat));
  float* st = stats.data_ptr<float>();
  const int64_t n_stat = (int64_t)d.B * d.N * d.Tq;
  c10::DeviceGuard guard(q.device());
  const int dt = dtype_code(q.scalar_type());
  int status;
  if (w.window) {
    const at::Tensor ws = w.workspace(q, d, causal);
    status = api().window_bwdbwd(current_stream(q), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                                 dout.data_ptr(), ddq.data_ptr(), ddk.data_ptr(), ddv.data_ptr(),
                                 lse.data_ptr<float>(), dq2.data_ptr(), dk2.data_ptr(), dv2.data_ptr(),
                                 ddo.data_ptr(), st, st + n_stat, st + 2 * n_stat, data_or_null(ws), d.B, d.Tq, d.Tk,
                                 d.N, d.Nk, d.H, dt, causal, w.window, w.sinks, (float)scale);
  } else {
    status = api().bwdbwd(current_stream(q), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                          dout.data_ptr(), ddq.data_ptr(), ddk.data_ptr(), ddv.data_ptr(), lse.data_ptr<float>(),
                          dq2.data_ptr(), dk2.data_ptr(), dv2.data_ptr(), ddo.data_ptr(), st, st + n_stat,
                          st + 2 * n_stat, d.B, d.Tq, d.Tk, d.N, d.Nk, d.H, dt, causal, (float)scale);
  }
  check_status(status);
  return {dq2, dk2, dv2, ddo, stats};
}

// -------------------------------------------------------------- paged cache

typedef c10::optional<at::Tensor> MaybeTensor;

const at::Tensor* get(const MaybeTensor& t) { return t && t->defined() ? &*t : nullptr; }
const void* ptr(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }

// Refuses an out whose memory a contiguous tensor that the kernels read shares; `same`: but for all
// of it, row by row.
void check_apart(const char* out_name, const at::Tensor& out, const char* name, const at::Tensor& t, bool same) {
  const char *a = (const char*)out.data_ptr(), *b = (const char*)t.data_ptr();
  if (a < b + t.nbytes() && b < a + out.nbytes() && !(same && a == b))
    value_error(std::string(out_name) + " overlaps " + name);
}

// A paged cache and what finds tokens in it, checked (_hip.py _check_cache).
struct Cache {
  const at::Tensor *k, *v, *k_scale = nullptr, *v_scale = nullptr;
  at::Tensor table, lengths, offsets;  // contiguous; offsets undefined if there are none
  int pages, kv_heads, page, head_dim, batch, width, dtype;

  Cache(const char* first_name, const at::Tensor& first, const at::Tensor& k_, const at::Tensor& v_,
        const at::Tensor& table_, const at::Tensor& lengths_, const MaybeTensor& offsets_, const MaybeTensor& ks,
        const MaybeTensor& vs, at::ScalarType dt)
      : k(&k_), v(&v_) {
    const bool quantised = k_.scalar_type() == at::kFloat8_e4m3fn;
    const at::Tensor *kst = get(ks), *vst = get(vs), *off = get(offsets_);
    check_inputs({{first_name, &first}, {"key_cache", &k_}, {"value_cache", &v_}, {"page_table", &table_},
                  {"lengths", &lengths_}},
                 c10::nullopt);
    if (quantised) {
      if (!kst || !vst) value_error("an e4m3 cache needs key_scale and value_scale");
      check_inputs({{first_name, &first}, {"key_scale", kst}, {"value_scale", vst}}, c10::nullopt);
    } else if (kst || vst) {
      value_error("key_scale and value_scale are for an e4m3 cache, not " + dtype_str(k_.scalar_type()));
    }
    if (off) check_inputs({{first_name, &first}, {"query_offsets", off}}, c10::nullopt);
    if (k_.dim() != 4) value_error("expected a (pages, kv_heads, page_size, head_dim) cache, got " + shape_str(k_));
    expect("value_cache", v_, k_.sizes(), k_.scalar_type());
    if (k_.scalar_type() != dt && !quantised)
      value_error("the cache must be of " + dtype_str(dt) + " or torch.float8_e4m3fn, got " +
                  dtype_str(k_.scalar_type()));
    if (!k_.is_contiguous()) value_error("key_cache must be contiguous");
    if (!v_.is_contiguous()) value_error("value_cache must be contiguous");
    if (quantised) {
      k_scale = kst;
      v_scale = vst;
      for (const auto& [name, t] : {std::pair<const char*, const at::Tensor*>{"key_scale", kst}, {"value_scale", vst}}) {
        expect(name, *t, k_.sizes().slice(0, 3));
        if ((t->scalar_type() != at::kFloat8_e8m0fnu && t->scalar_type() != at::kByte) || !t->is_contiguous())
          value_error(std::string(name) + " must be a contiguous tensor of torch.float8_e8m0fnu or torch.uint8");
      }
    }
    if (table_.dim() != 2) value_error("expected a (batch, pages) page_table, got " + shape_str(table_));
    expect("lengths", lengths_, {table_.size(0)});
    if (off) expect("query_offsets", *off, {table_.size(0) + 1});
    for (const auto& [name, t] : {std::pair<const char*, const at::Tensor*>{"page_table", &table_},
                                  {"lengths", &lengths_}, {"query_offsets", off}})
      if (t && t->scalar_type() != at::kInt)
        value_error(std::string(name) + " has dtype " + dtype_str(t->scalar_type()) + ", expected torch.int32");
    for (int64_t s : k_.sizes())
      if (s > INT32_MAX) value_error("key_cache" + shape_str(k_) + " has a dimension beyond the C ABI's int range");
    for (int64_t s : table_.sizes())
      if (s > INT32_MAX) value_error("page_table" + shape_str(table_) + " has a dimension beyond the C ABI's int range");
    table = contig(table_);
    lengths = contig(lengths_);
    if (off) offsets = contig(*off);
    pages = (int)k_.size(0), kv_heads = (int)k_.size(1), page = (int)k_.size(2), head_dim = (int)k_.size(3);
    batch = (int)table_.size(0), width = (int)table_.size(1);
    dtype = quantised ? FHOG_DTYPE_E4M3 : dtype_code(dt);
  }
  // Refuses an out that shares memory with any of it.
  void check_apart_from(const char* out_name, const at::Tensor& out) const {
    for (const auto& [name, t] : {std::pair<const char*, const at::Tensor*>{"key_cache", k}, {"value_cache", v},
                                  {"key_scale", k_scale}, {"value_scale", v_scale}, {"page_table", &table},
                                  {"lengths", &lengths}, {"query_offsets", offsets.defined() ? &offsets : nullptr}})
      if (t) check_apart(out_name, out, name, *t, false);
  }
  const int* table_ptr() const { return table.data_ptr<int>(); }
  const int* lengths_ptr() const { return lengths.data_ptr<int>(); }
  const int* offsets_ptr() const { return offsets.defined() ? offsets.data_ptr<int>() : nullptr; }
};

// Tells autograd that a tensor was written to: a graph that saved it before then raises in its
// backward. (Inference tensors, which no graph can save, have no version.)
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

int rows_of(const char* name, const at::Tensor& t) {
  if (t.dim() != 3) value_error(std::string("expected a (T, N, H) ") + name + ", got " + shape_str(t));
  for (int64_t s : t.sizes())
    if (s > INT32_MAX) value_error(name + shape_str(t) + " has a dimension beyond the C ABI's int range");
  return (int)t.size(0);
}

at::Tensor paged_attention_core(const at::Tensor& q_, const at::Tensor& k_cache, const at::Tensor& v_cache,
                                const at::Tensor& table, const at::Tensor& lengths, const MaybeTensor& offsets,
                                const MaybeTensor& k_scale, const MaybeTensor& v_scale, int window, int sinks,
                                double scale, const MaybeTensor& out_) {
  const int total = rows_of("query", q_);
  const Cache c("query", q_, k_cache, v_cache, table, lengths, offsets, k_scale, v_scale, q_.scalar_type());
  if (q_.size(2) != c.head_dim)
    value_error("query" + shape_str(q_) + " and key_cache" + shape_str(k_cache) + " disagree on head_dim");
  const int dt = dtype_code(q_.scalar_type());
  const at::Tensor* given = get(out_);
  if (given) {
    check_inputs({{"query", &q_}, {"out", given}}, q_.scalar_type());
    expect("out", *given, q_.sizes());
    if (!given->is_contiguous()) value_error("out must be contiguous");
  }
  at::Tensor out = given ? *given : at::empty(q_.sizes(), q_.options());
  const at::Tensor q = contig(q_);
  if (given) {
    check_apart("out", out, "query", q, true);
    c.check_apart_from("out", out);
  }
  const int heads = (int)q.size(1);
  c10::DeviceGuard guard(q.device());
  const size_t size = api().paged_bytes(c.batch, total, !c.offsets.defined(), heads, c.kv_heads, c.head_dim, c.page,
                                        c.width, window, sinks);
  const at::Tensor ws = size ? at::empty({(int64_t)size}, q.options().dtype(at::kByte)) : at::Tensor();
  check_status(api().paged_attention(current_stream(q), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                     ptr(c.k_scale), ptr(c.v_scale), c.table_ptr(), c.lengths_ptr(), c.offsets_ptr(),
                                     out.data_ptr(), data_or_null(ws), size, c.batch, total, heads, c.kv_heads,
                                     c.head_dim, c.pages, c.page, c.width, dt, c.dtype, window, sinks, given == nullptr,
                                     (float)scale));
  if (given) written(out);
  return out;
}

void cache_write_core(const at::Tensor& k_, const at::Tensor& v_, const at::Tensor& k_cache, const at::Tensor& v_cache,
                      const at::Tensor& table, const at::Tensor& lengths, const MaybeTensor& offsets,
                      const MaybeTensor& k_scale, const MaybeTensor& v_scale) {
  const int total = rows_of("key", k_);
  const Cache c("key", k_, k_cache, v_cache, table, lengths, offsets, k_scale, v_scale, k_.scalar_type());
  check_inputs({{"key", &k_}, {"value", &v_}}, k_.scalar_type());
  expect("value", v_, k_.sizes());
  if (k_.size(1) != c.kv_heads || k_.size(2) != c.head_dim)
    value_error("key" + shape_str(k_) + " and key_cache" + shape_str(k_cache) + " disagree on heads or head_dim");
  const int dt = dtype_code(k_.scalar_type());
  const at::Tensor k = contig(k_), v = contig(v_);
  c10::DeviceGuard guard(k.device());
  check_status(api().cache_write(current_stream(k), k.data_ptr(), v.data_ptr(), k_cache.data_ptr(),
                                 v_cache.data_ptr(), const_cast<void*>(ptr(c.k_scale)),
                                 const_cast<void*>(ptr(c.v_scale)), c.table_ptr(), c.lengths_ptr(), c.offsets_ptr(),
                                 c.batch, total, c.kv_heads, c.head_dim, c.pages, c.page, c.width, dt, c.dtype));
  for (const at::Tensor* t : {&k_cache, &v_cache, c.k_scale, c.v_scale})
    if (t) written(*t);
}

std::tuple<at::Tensor, at::Tensor> cache_read_core(const at::Tensor& k_cache, const at::Tensor& v_cache,
                                                   const at::Tensor& table, const at::Tensor& lengths,
                                                   int64_t max_length, at::ScalarType dtype,
                                                   const MaybeTensor& k_scale, const MaybeTensor& v_scale) {
  const Cache c("key_cache", k_cache, k_cache, v_cache, table, lengths, c10::nullopt, k_scale, v_scale, dtype);
  if (max_length < 0) value_error("max_length must be >= 0, got " + std::to_string(max_length));
  if (max_length > INT32_MAX) value_error("max_length is beyond the C ABI's int range");
  const int dt = dtype_code(dtype);
  const auto options = k_cache.options().dtype(dtype);
  at::Tensor k = at::empty({(int64_t)c.batch, max_length, (int64_t)c.kv_heads, (int64_t)c.head_dim}, options);
  at::Tensor v = at::empty(k.sizes(), options);
  c10::DeviceGuard guard(k.device());
  check_status(api().cache_read(current_stream(k), k_cache.data_ptr(), v_cache.data_ptr(), ptr(c.k_scale),
                                ptr(c.v_scale), c.table_ptr(), c.lengths_ptr(), k.data_ptr(), v.data_ptr(), c.batch,
                                (int)max_length, c.kv_heads, c.head_dim, c.pages, c.page, c.width, dt, c.dtype));
  return {k, v};
}

// ------------------------------------------------- the cache's allocator, chosen blocks

bool overlap(const at::Tensor& x, const at::Tensor& y) {
  const char *a = (const char*)x.data_ptr(), *b = (const char*)y.data_ptr();
  return a < b + y.nbytes() && b < a + x.nbytes();
}

at::Tensor bytes_on(const at::Tensor& like, size_t size) {
  return size ? at::empty({(int64_t)size}, like.options().dtype(at::kByte)) : at::Tensor();
}

at::Tensor cache_extend_core(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& table,
                             const at::Tensor& lengths, const MaybeTensor& new_tokens, int new_each,
                             const MaybeTensor& parents, const MaybeTensor& k_scale, const MaybeTensor& v_scale) {
  const Cache c("key_cache", k_cache, k_cache, v_cache, table, lengths, c10::nullopt, k_scale, v_scale,
                k_cache.scalar_type());
  for (const auto& [name, t] : {std::pair<const char*, const at::Tensor*>{"page_table", &table}, {"lengths", &lengths}})
    if (!t->is_contiguous()) value_error(std::string(name) + " must be contiguous");
  at::Tensor held[2];  // parents, new_tokens
  int i = 0;
  for (const auto& [name, t] : {std::pair<const char*, const at::Tensor*>{"parents", get(parents)},
                                {"new_tokens", get(new_tokens)}}) {
    at::Tensor& to = held[i++];
    if (!t) continue;
    check_inputs({{"key_cache", &k_cache}, {name, t}}, c10::nullopt);
    expect(name, *t, {table.size(0)}, at::kInt);
    if (overlap(*t, table) || overlap(*t, lengths))
      value_error(std::string(name) + " overlaps page_table or lengths");
    to = contig(*t);
  }
  if (c.batch == 0) value_error("expected at least one row of page_table");
  at::Tensor free = at::empty({}, lengths.options());
  c10::DeviceGuard guard(k_cache.device());
  const size_t size = api().pages_bytes(c.batch, c.pages, c.width);
  const at::Tensor ws = bytes_on(k_cache, size);
  check_status(api().cache_extend(current_stream(k_cache), k_cache.data_ptr(), v_cache.data_ptr(),
                                  const_cast<void*>(ptr(c.k_scale)), const_cast<void*>(ptr(c.v_scale)),
                                  table.data_ptr<int>(), lengths.data_ptr<int>(), (const int*)data_or_null(held[0]),
                                  (const int*)data_or_null(held[1]), new_each, free.data_ptr<int>(), data_or_null(ws), size,
                                  c.batch, c.kv_heads, c.head_dim, c.pages, c.page, c.width, c.dtype));
  for (const at::Tensor* t : {&k_cache, &v_cache, c.k_scale, c.v_scale, &table, &lengths})
    if (t) written(*t);
  return free;
}

void check_key_means(const at::Tensor& means, const char* first_name, const at::Tensor& first, at::IntArrayRef shape) {
  check_inputs({{first_name, &first}, {"key_means", &means}}, c10::nullopt);
  expect("key_means", means, shape, at::kFloat);
  if (!means.is_contiguous()) value_error("key_means must be contiguous");
}

// (k_cache, v_cache, k_scale, v_scale, key_means, page_table), undefined for what is not given.
std::tuple<at::Tensor, at::Tensor, MaybeTensor, MaybeTensor, MaybeTensor, at::Tensor> cache_compact_core(
    const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& table, const at::Tensor& lengths,
    int64_t num_pages, const MaybeTensor& k_scale, const MaybeTensor& v_scale, const MaybeTensor& key_means) {
  const Cache c("key_cache", k_cache, k_cache, v_cache, table, lengths, c10::nullopt, k_scale, v_scale,
                k_cache.scalar_type());
  const at::Tensor* means = get(key_means);
  if (means) check_key_means(*means, "key_cache", k_cache, {k_cache.size(0), k_cache.size(1), k_cache.size(3)});
  if (num_pages < 1 || num_pages > INT32_MAX)
    value_error("num_pages must be >= 1 and below 2 ** 31, got " + std::to_string(num_pages));
  const at::Tensor* in[5] = {&k_cache, &v_cache, c.k_scale, c.v_scale, means};
  at::Tensor out[5];
  for (int i = 0; i < 5; ++i)
    if (in[i]) {
      std::vector<int64_t> shape = in[i]->sizes().vec();
      shape[0] = num_pages;
      out[i] = at::empty(shape, in[i]->options());
    }
  at::Tensor table_out = at::empty(table.sizes(), table.options());
  c10::DeviceGuard guard(k_cache.device());
  const size_t size = api().pages_bytes(c.batch, c.pages, c.width);
  const at::Tensor ws = bytes_on(k_cache, size);
  check_status(api().cache_compact(
      current_stream(k_cache), k_cache.data_ptr(), v_cache.data_ptr(), ptr(c.k_scale), ptr(c.v_scale), (const float*)ptr(means),
      c.table_ptr(), c.lengths_ptr(), out[0].data_ptr(), out[1].data_ptr(), data_or_null(out[2]), data_or_null(out[3]),
      (float*)data_or_null(out[4]), table_out.data_ptr<int>(), data_or_null(ws), size, c.batch, c.kv_heads, c.head_dim, c.pages,
      c.page, c.width, (int)num_pages, c.dtype));
  auto maybe = [](const at::Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); };  // None in Python
  return {out[0], out[1], maybe(out[2]), maybe(out[3]), maybe(out[4]), table_out};
}

void key_means_core(const at::Tensor& k_cache, const at::Tensor& means, const at::Tensor& table, const at::Tensor& lengths,
                    const MaybeTensor& offsets, const MaybeTensor& k_scale) {
  const Cache c("key_cache", k_cache, k_cache, k_cache, table, lengths, offsets, k_scale, k_scale, k_cache.scalar_type());
  check_key_means(means, "key_cache", k_cache, {k_cache.size(0), k_cache.size(1), k_cache.size(3)});
  c.check_apart_from("key_means", means);
  c10::DeviceGuard guard(k_cache.device());
  check_status(api().key_means(current_stream(k_cache), k_cache.data_ptr(), ptr(c.k_scale), means.data_ptr<float>(),
                               c.table_ptr(), c.lengths_ptr(), c.offsets_ptr(), c.batch, c.kv_heads, c.head_dim, c.pages,
                               c.page, c.width, c.dtype));
  written(means);
}

at::Tensor block_select_core(const at::Tensor& q_, const at::Tensor& means, const at::Tensor& table,
                             const at::Tensor& lengths, const MaybeTensor& offsets_, int64_t page_size, int64_t blocks,
                             int64_t first, int64_t last) {
  const int total = rows_of("query", q_);
  if (means.dim() != 3 || means.size(2) != q_.size(2))
    value_error("expected (pages, kv_heads, head_dim) key_means for query" + shape_str(q_) + ", got " + shape_str(means));
  check_key_means(means, "query", q_, means.sizes());
  const at::Tensor* off = get(offsets_);
  check_inputs({{"query", &q_}, {"page_table", &table}, {"lengths", &lengths}}, c10::nullopt);
  if (off) check_inputs({{"query", &q_}, {"query_offsets", off}}, c10::nullopt);
  if (table.dim() != 2) value_error("expected a (batch, pages) page_table, got " + shape_str(table));
  expect("lengths", lengths, {table.size(0)});
  if (off) expect("query_offsets", *off, {table.size(0) + 1});
  for (const auto& [name, t] : {std::pair<const char*, const at::Tensor*>{"page_table", &table},
                                {"lengths", &lengths}, {"query_offsets", off}})
    if (t && t->scalar_type() != at::kInt)
      value_error(std::string(name) + " has dtype " + dtype_str(t->scalar_type()) + ", expected torch.int32");
  const int dt = dtype_code(q_.scalar_type());
  for (int64_t s : {means.size(0), means.size(1), table.size(0), table.size(1), page_size})
    if (s > INT32_MAX) value_error("a size is beyond the C ABI's int range");
  if (blocks < 1 || blocks > 32768) value_error("blocks must be 1 to 32768, got " + std::to_string(blocks));
  if (first < 0 || last < 1 || first + last > blocks)
    value_error("needs first >= 0, last >= 1 and first + last <= blocks, got " + std::to_string(first) + ", " +
                std::to_string(last) + " and " + std::to_string(blocks));
  const at::Tensor q = contig(q_), t = contig(table), n = contig(lengths), o = off ? contig(*off) : at::Tensor();
  const int kv = (int)means.size(1), batch = (int)table.size(0), width = (int)table.size(1);
  at::Tensor chosen = at::empty({(int64_t)total, (int64_t)kv, blocks}, t.options());
  c10::DeviceGuard guard(q.device());
  const size_t size = api().select_bytes(batch, total, !off, kv, (int)q.size(2), width, (int)first, (int)last);
  const at::Tensor ws = bytes_on(q, size);
  check_status(api().block_select(current_stream(q), q.data_ptr(), means.data_ptr<float>(), t.data_ptr<int>(),
                                  n.data_ptr<int>(), (const int*)data_or_null(o), chosen.data_ptr<int>(), data_or_null(ws),
                                  size, batch, total, (int)q.size(1), kv, (int)q.size(2), (int)means.size(0), (int)page_size,
                                  width, dt, (int)blocks, (int)first, (int)last));
  return chosen;
}

at::Tensor block_attention_core(const at::Tensor& q_, const at::Tensor& chosen_, const at::Tensor& k_cache,
                                const at::Tensor& v_cache, const at::Tensor& table, const at::Tensor& lengths,
                                const MaybeTensor& offsets, const MaybeTensor& k_scale, const MaybeTensor& v_scale,
                                double scale, const MaybeTensor& out_) {
  const int total = rows_of("query", q_);
  const Cache c("query", q_, k_cache, v_cache, table, lengths, offsets, k_scale, v_scale, q_.scalar_type());
  if (q_.size(2) != c.head_dim)
    value_error("query" + shape_str(q_) + " and key_cache" + shape_str(k_cache) + " disagree on head_dim");
  const int dt = dtype_code(q_.scalar_type());
  check_inputs({{"query", &q_}, {"blocks", &chosen_}}, c10::nullopt);
  if (chosen_.dim() != 3 || chosen_.size(0) != total || chosen_.size(1) != c.kv_heads || chosen_.scalar_type() != at::kInt)
    value_error("blocks must be torch.int32 (" + std::to_string(total) + ", " + std::to_string(c.kv_heads) +
                ", 'blocks'), got " + shape_str(chosen_) + " of " + dtype_str(chosen_.scalar_type()));
  if (chosen_.size(2) > INT32_MAX) value_error("blocks has a dimension beyond the C ABI's int range");
  const at::Tensor* given = get(out_);
  if (given) {
    check_inputs({{"query", &q_}, {"out", given}}, q_.scalar_type());
    expect("out", *given, q_.sizes());
    if (!given->is_contiguous()) value_error("out must be contiguous");
  }
  at::Tensor out = given ? *given : at::empty(q_.sizes(), q_.options());
  const at::Tensor q = contig(q_), chosen = contig(chosen_);
  if (given) {
    check_apart("out", out, "query", q, false);
    check_apart("out", out, "blocks", chosen, false);
    c.check_apart_from("out", out);
  }
  const int heads = (int)q.size(1), blocks = (int)chosen.size(2), single = !c.offsets.defined();
  c10::DeviceGuard guard(q.device());
  const size_t size = api().block_bytes(c.batch, total, single, heads, c.kv_heads, c.head_dim, c.page, c.width, blocks);
  const at::Tensor ws = bytes_on(q, size);
  check_status(api().block_attention(current_stream(q), q.data_ptr(), chosen.data_ptr<int>(), k_cache.data_ptr(),
                                     v_cache.data_ptr(), ptr(c.k_scale), ptr(c.v_scale), c.table_ptr(), c.lengths_ptr(),
                                     c.offsets_ptr(), out.data_ptr(), data_or_null(ws), size, c.batch, total, heads,
                                     c.kv_heads, c.head_dim, c.pages, c.page, c.width, dt, c.dtype, blocks,
                                     given == nullptr, (float)scale));
  if (given) written(out);
  return out;
}

// ------------------------------------------------- norms with rotation

// What the three calls share, checked (_hip.py _RotaryCall); q and k of three axes are unbatched. Where the rows are
// not read (`rows` false), q and k only give their shapes.
struct RotaryOptions {
  bool interleaved;
  c10::optional<double> eps;
};
struct RotaryWhere {
  at::Tensor frequencies, positions, lengths, offsets;  // undefined: none
};
struct RotaryCall {
  at::Tensor q, k, wq, wk;
  RotaryWhere at;
  fhog_rotary shape{};

  RotaryCall(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& wq_, const at::Tensor& wk_,
             const RotaryWhere& where, const RotaryOptions& o, bool rows) {
    check_inputs({{"query", &q_}, {"key", &k_}}, c10::nullopt);
    for (const auto& [name, t] : {std::pair<const char*, const at::Tensor*>{"query_weight", &wq_}, {"key_weight", &wk_},
                                  {"frequencies", &where.frequencies}, {"positions", &where.positions},
                                  {"lengths", &where.lengths}, {"query_offsets", &where.offsets}})
      if (t->defined()) check_inputs({{"query", &q_}, {name, t}}, c10::nullopt);
    check_inputs({{"query", &q_}, {"key", &k_}}, q_.scalar_type());
    const int dt = dtype_code(q_.scalar_type());
    const int64_t d = q_.dim();
    if ((d != 3 && d != 4) || k_.dim() != d || q_.size(0) != k_.size(0) || (d == 4 && q_.size(1) != k_.size(1)) ||
        q_.size(d - 1) != k_.size(d - 1))
      value_error("expected query (B, T, N, H) and key (B, T, N_kv, H) of the same tokens and head_dim, got " +
                  shape_str(q_) + " and " + shape_str(k_));
    const int64_t B = d == 4 ? q_.size(0) : 1, T = q_.size(d - 3), H = q_.size(d - 1);
    for (int64_t s : {B, T, q_.size(d - 2), k_.size(d - 2), H})
      if (s > INT32_MAX) value_error("query" + shape_str(q_) + " has a dimension beyond the C ABI's int range");
    if (!o.eps && (wq_.defined() || wk_.defined())) value_error("weights need norms (eps is None)");
    const at::ScalarType wt = wq_.defined() ? wq_.scalar_type() : wk_.defined() ? wk_.scalar_type() : q_.scalar_type();
    if (wq_.defined()) expect("query_weight", wq_, {H}, wt);
    if (wk_.defined()) expect("key_weight", wk_, {H}, wt);
    if (wt != q_.scalar_type() && wt != at::kFloat)
      value_error("weights must be of " + dtype_str(q_.scalar_type()) + " or torch.float32, got " + dtype_str(wt));
    const at::Tensor &f = where.frequencies, &p = where.positions, &n = where.lengths, &off = where.offsets;
    if (f.defined() && (f.dim() != 1 || 2 * f.size(0) > H || f.scalar_type() != at::kFloat))
      value_error("frequencies must be torch.float32 (R / 2,) with R <= head_dim, got " + shape_str(f) + " of " +
                  dtype_str(f.scalar_type()) + " for head_dim " + std::to_string(H));
    if (p.defined()) {
      if (n.defined()) value_error("positions and lengths exclude each other");
      if (p.scalar_type() != at::kInt && p.scalar_type() != at::kLong)
        value_error("positions has dtype " + dtype_str(p.scalar_type()) + ", expected torch.int32 or torch.int64");
      if (!(p.dim() == 1 && p.size(0) == T) && !(p.dim() == 2 && p.size(0) == B && p.size(1) == T))
        value_error("positions has shape " + shape_str(p) + ", expected (" + std::to_string(T) + ",) or (" +
                    std::to_string(B) + ", " + std::to_string(T) + ")");
    }
    if (off.defined() && !n.defined()) value_error("query_offsets needs lengths");
    if (n.defined()) {
      if (n.dim() != 1) value_error("expected (batch,) lengths, got " + shape_str(n));
      if (B != 1) value_error("lengths go with packed tokens (T, N, H), got a batch of " + std::to_string(B));
      if (off.defined())
        expect("query_offsets", off, {n.size(0) + 1});
      else
        expect("lengths", n, {T});
      for (const auto& [name, t] : {std::pair<const char*, const at::Tensor*>{"lengths", &n}, {"query_offsets", &off}})
        if (t->defined() && t->scalar_type() != at::kInt)
          value_error(std::string(name) + " has dtype " + dtype_str(t->scalar_type()) + ", expected torch.int32");
    }
    auto lines = [&](const at::Tensor& t) { return !rows || t.stride(d - 1) == 1 || H == 1 ? t : t.contiguous(); };
    q = lines(q_), k = lines(k_);
    auto held = [](const at::Tensor& t) { return t.defined() ? contig(t) : t; };
    wq = held(wq_), wk = held(wk_);
    at = {held(f), held(p), held(n), held(off)};
    shape.batch = (int)B, shape.tokens = (int)T, shape.heads = (int)q.size(d - 2), shape.kv_heads = (int)k.size(d - 2);
    shape.head_dim = (int)H, shape.rotated = f.defined() ? 2 * (int)f.size(0) : 0;
    shape.dtype = dt, shape.weight_dtype = dtype_code(wt);
    shape.interleaved = o.interleaved, shape.norm = o.eps.has_value(), shape.eps = o.eps ? (float)*o.eps : 0.f;
    shape.position_bytes = p.defined() ? (int)p.element_size() : 0;
    shape.position_rows = !p.defined() ? 0 : p.dim() == 1 ? 1 : (int)B;
    shape.sequences = n.defined() ? (int)n.size(0) : 0;
    for (int i = 0; i < 3; ++i) {
      const int64_t axis = i + d - 4;
      shape.q_stride[i] = axis < 0 ? 0 : q.stride(axis);
      shape.k_stride[i] = axis < 0 ? 0 : k.stride(axis);
    }
    shape.frequencies = (const float*)data_or_null(at.frequencies);
    shape.positions = data_or_null(at.positions);
    shape.lengths = (const int*)data_or_null(at.lengths);
    shape.query_offsets = (const int*)data_or_null(at.offsets);
  }
  at::Tensor like(const at::Tensor& t) const { return at::empty(t.sizes(), t.options()); }
  at::Tensor like_weight(const at::Tensor& w) const { return w.defined() ? at::empty(w.sizes(), w.options()) : w; }
  // A tensor of q's (or k's) shape, contiguous.
  at::Tensor rows(const char* name, const at::Tensor& t, const at::Tensor& x) const {
    check_inputs({{"query", &q}, {name, &t}}, q.scalar_type());
    expect(name, t, x.sizes());
    return contig(t);
  }
  at::Tensor workspace() const {
    return wq.defined() || wk.defined() ? bytes_on(q, api().rotary_bytes(&shape)) : at::Tensor();
  }
};

std::tuple<at::Tensor, at::Tensor> rotary_fwd_core(const at::Tensor& q, const at::Tensor& k, const at::Tensor& wq,
                                                   const at::Tensor& wk, const RotaryWhere& where,
                                                   const RotaryOptions& o) {
  const RotaryCall c(q, k, wq, wk, where, o, true);
  at::Tensor q_out = c.like(c.q), k_out = c.like(c.k);
  c10::DeviceGuard guard(c.q.device());
  check_status(api().rotary_fwd(current_stream(c.q), &c.shape, c.q.data_ptr(), c.k.data_ptr(), data_or_null(c.wq),
                                data_or_null(c.wk), q_out.data_ptr(), k_out.data_ptr()));
  return {q_out, k_out};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> rotary_bwd_core(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& wq, const at::Tensor& wk, const at::Tensor& gq_,
    const at::Tensor& gk_, const RotaryWhere& where, const RotaryOptions& o) {
  const RotaryCall c(q, k, wq, wk, where, o, o.eps.has_value());
  const at::Tensor gq = c.rows("query's cotangent", gq_, c.q), gk = c.rows("key's cotangent", gk_, c.k);
  at::Tensor dq = c.like(c.q), dk = c.like(c.k), dwq = c.like_weight(c.wq), dwk = c.like_weight(c.wk);
  c10::DeviceGuard guard(c.q.device());
  const at::Tensor ws = c.workspace();
  check_status(api().rotary_bwd(current_stream(c.q), &c.shape, o.eps ? c.q.data_ptr() : nullptr,
                                o.eps ? c.k.data_ptr() : nullptr, data_or_null(c.wq), data_or_null(c.wk), gq.data_ptr(),
                                gk.data_ptr(), dq.data_ptr(), dk.data_ptr(), data_or_null(dwq), data_or_null(dwk),
                                data_or_null(ws)));
  return {dq, dk, dwq, dwk};
}

// dq2, dk2, dwq2, dwk2, dgq, dgk
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> rotary_bwdbwd_core(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& wq, const at::Tensor& wk, const at::Tensor& gq_,
    const at::Tensor& gk_, const at::Tensor& uq_, const at::Tensor& uk_, const at::Tensor& zq_, const at::Tensor& zk_,
    const RotaryWhere& where, const RotaryOptions& o) {
  const RotaryCall c(q, k, wq, wk, where, o, true);
  const at::Tensor gq = c.rows("query's cotangent", gq_, c.q), gk = c.rows("key's cotangent", gk_, c.k);
  const at::Tensor uq = c.rows("cotangent of query's gradient", uq_, c.q), uk = c.rows("cotangent of key's gradient", uk_, c.k);
  auto weight = [&](const at::Tensor& w, const at::Tensor& z) {
    if (!w.defined()) return at::Tensor();
    check_inputs({{"query", &c.q}, {"cotangent of a weight's gradient", &z}}, c10::nullopt);
    expect("cotangent of a weight's gradient", z, w.sizes(), w.scalar_type());
    return contig(z);
  };
  const at::Tensor zq = weight(c.wq, zq_), zk = weight(c.wk, zk_);
  at::Tensor dq2 = c.like(c.q), dk2 = c.like(c.k), dgq = c.like(c.q), dgk = c.like(c.k);
  at::Tensor dwq2 = c.like_weight(c.wq), dwk2 = c.like_weight(c.wk);
  c10::DeviceGuard guard(c.q.device());
  const at::Tensor ws = c.workspace();
  check_status(api().rotary_bwdbwd(current_stream(c.q), &c.shape, c.q.data_ptr(), c.k.data_ptr(), data_or_null(c.wq),
                                   data_or_null(c.wk), gq.data_ptr(), gk.data_ptr(), uq.data_ptr(), uk.data_ptr(),
                                   data_or_null(zq), data_or_null(zk), dq2.data_ptr(), dk2.data_ptr(), data_or_null(dwq2),
                                   data_or_null(dwk2), dgq.data_ptr(), dgk.data_ptr(), data_or_null(ws)));
  return {dq2, dk2, dwq2, dwk2, dgq, dgk};
}

// ------------------------------------------------------------------ autograd

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Refuses a third derivative as the once_differentiable double backward of
// flash_hog/torch/attention.py does. Under create_graph, with cotangents that
// require grad, the double backward's results are detached, marked as
// requiring grad and passed through this node (as copies), whose backward
// raises: a backward() through them raises, while a grad() with respect to
// the inputs finds no path through them.
struct NoThirdOrder : public torch::autograd::Function<NoThirdOrder> {
  static variable_list forward(AutogradContext*, const at::Tensor& dq2, const at::Tensor& dk2,
                               const at::Tensor& dv2, const at::Tensor& ddo) {
    return {dq2.clone(), dk2.clone(), dv2.clone(), ddo.clone()};
  }
  static variable_list backward(AutogradContext*, variable_list) {
    throw std::runtime_error("trying to differentiate twice a function that was marked with @once_differentiable");
  }
};

// A call's mask and scale, as one argument of the Functions.
struct Mask {
  int causal;
  double scale;
  Window w;
  void save(AutogradContext* ctx) const {
    ctx->saved_data["causal"] = (int64_t)causal;
    ctx->saved_data["scale"] = scale;
    if (w.window == 0) return;  // (an entry costs every call)
    ctx->saved_data["window"] = (int64_t)w.window;
    ctx->saved_data["sinks"] = (int64_t)w.sinks;
  }
  static Mask saved(AutogradContext* ctx) {
    Mask m{(int)ctx->saved_data["causal"].toInt(), ctx->saved_data["scale"].toDouble(), {}};
    const auto window = ctx->saved_data.find("window");
    if (window != ctx->saved_data.end())
      m.w = {(int)window->second.toInt(), (int)ctx->saved_data["sinks"].toInt()};
    return m;
  }
};

// Primal (q, k, v, O, L, dO) -> (dQ, dK, dV), differentiable once in q, k, v
// and dO: _DotProductAttentionBwd (the rule
// dot_product_attention_bwd_rule_fwd_rule and its rule
// dot_product_attention_bwd_rule_bwd_rule).
struct AttentionBwdFn : public torch::autograd::Function<AttentionBwdFn> {
  static variable_list forward(AutogradContext* ctx, const Mask& mask, const at::Tensor& q, const at::Tensor& k,
                               const at::Tensor& v, const at::Tensor& lse, const at::Tensor& o, const at::Tensor& g) {
    auto [dq, dk, dv, delta] = bwd_core(q, k, v, o, g, lse, mask.causal, mask.scale, mask.w);
    ctx->save_for_backward({q, k, v, o, lse, g});
    mask.save(ctx);
    return {dq, dk, dv};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list r = ctx->get_saved_variables();  // q, k, v, O, L, dO
    const Mask mask = Mask::saved(ctx);
    auto [dq2, dk2, dv2, ddo, stats] = bwdbwd_core(r[0], r[1], r[2], r[3], r[5], grads[0], grads[1], grads[2], r[4],
                                                   mask.causal, mask.scale, mask.w);
    if (c10::GradMode::is_enabled() &&
        (grads[0].requires_grad() || grads[1].requires_grad() || grads[2].requires_grad())) {
      auto mark = [](const at::Tensor& t) { return t.detach().requires_grad_(true); };
      const variable_list w = NoThirdOrder::apply(mark(dq2), mark(dk2), mark(dv2), mark(ddo));
      dq2 = w[0], dk2 = w[1], dv2 = w[2], ddo = w[3];
    }
    // no cotangent for L and O (flash_hog/jax/_attention_impl.py:278-303)
    return {at::Tensor(), dq2, dk2, dv2, at::Tensor(), at::Tensor(), ddo};
  }
};

// Primal (q, k, v) -> (O, L), L not differentiable: _DotProductAttention (the
// rule dot_product_attention_fwd_rule and its rule
// dot_product_attention_bwd_rule, through AttentionBwdFn).
struct AttentionFn : public torch::autograd::Function<AttentionFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                               const Mask& mask) {
    auto [o, lse] = fwd_core(q, k, v, mask.causal, mask.scale, mask.w);
    ctx->save_for_backward({q, k, v, lse, o});
    mask.save(ctx);
    ctx->mark_non_differentiable({lse});
    return {o, lse};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list r = ctx->get_saved_variables();  // q, k, v, L, O
    // O enters the first backward as a constant: the double backward returns
    // no cotangent for it, and detaching it keeps this node out of a second
    // derivative's graph.
    const variable_list d = AttentionBwdFn::apply(Mask::saved(ctx), r[0], r[1], r[2], r[3], r[4].detach(), grads[0]);
    return {d[0], d[1], d[2], at::Tensor()};
  }
};

// qk_norm_rotary's nodes, as flash_hog/torch/rotary.py has them. Absent tensors are undefined, among the nodes'
// arguments (which take no undefined ones) empty; a result that an absent weight would have is a tensor of no
// elements.
at::Tensor given(const MaybeTensor& t) { return t ? *t : at::Tensor(); }
MaybeTensor maybe(const at::Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }

struct RotarySaved {
  static void save(AutogradContext* ctx, const RotaryWhere& w, const RotaryOptions& o, variable_list more) {
    variable_list all = {w.frequencies, w.positions, w.lengths, w.offsets};
    all.insert(all.end(), more.begin(), more.end());
    ctx->save_for_backward(std::move(all));
    ctx->saved_data["interleaved"] = o.interleaved;
    if (o.eps) ctx->saved_data["eps"] = *o.eps;
  }
  static RotaryOptions options(AutogradContext* ctx) {
    const auto eps = ctx->saved_data.find("eps");
    return {ctx->saved_data["interleaved"].toBool(),
            eps == ctx->saved_data.end() ? c10::nullopt : c10::optional<double>(eps->second.toDouble())};
  }
  static RotaryWhere where(const variable_list& r) { return {r[0], r[1], r[2], r[3]}; }
};

// Refuses a third derivative (NoThirdOrder).
struct NoThirdOrderRotary : public torch::autograd::Function<NoThirdOrderRotary> {
  static variable_list forward(AutogradContext*, const at::Tensor& a, const at::Tensor& b, const at::Tensor& c,
                               const at::Tensor& d, const at::Tensor& e, const at::Tensor& f) {
    return {a.clone(), b.clone(), c.clone(), d.clone(), e.clone(), f.clone()};
  }
  static variable_list backward(AutogradContext*, variable_list) {
    throw std::runtime_error("trying to differentiate twice a function that was marked with @once_differentiable");
  }
};

struct RotaryBwdFn : public torch::autograd::Function<RotaryBwdFn> {
  static variable_list forward(AutogradContext* ctx, const RotaryOptions& o, const at::Tensor& q, const at::Tensor& k,
                               const MaybeTensor& wq_, const MaybeTensor& wk_, const at::Tensor& gq, const at::Tensor& gk,
                               const MaybeTensor& frequencies, const MaybeTensor& positions, const MaybeTensor& lengths,
                               const MaybeTensor& offsets) {
    const at::Tensor wq = given(wq_), wk = given(wk_);
    const RotaryWhere w{given(frequencies), given(positions), given(lengths), given(offsets)};
    auto [dq, dk, dwq, dwk] = rotary_bwd_core(q, k, wq, wk, gq, gk, w, o);
    RotarySaved::save(ctx, w, o, o.eps ? variable_list{q, k, wq, wk, gq, gk} : variable_list{});
    if (!dwq.defined()) dwq = at::empty({0}, q.options());
    if (!dwk.defined()) dwk = at::empty({0}, k.options());
    return {dq, dk, dwq, dwk};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list r = ctx->get_saved_variables();
    const RotaryOptions o = RotarySaved::options(ctx);
    const RotaryWhere w = RotarySaved::where(r);
    at::Tensor none, d[6];  // dq2, dk2, dwq2, dwk2, dgq, dgk
    if (o.eps)
      std::tie(d[0], d[1], d[2], d[3], d[4], d[5]) =
          rotary_bwdbwd_core(r[4], r[5], r[6], r[7], r[8], r[9], grads[0], grads[1], grads[2], grads[3], w, o);
    else
      std::tie(d[4], d[5]) = rotary_fwd_core(grads[0], grads[1], none, none, w, o);
    if (c10::GradMode::is_enabled() &&
        std::any_of(grads.begin(), grads.end(), [](const at::Tensor& t) { return t.requires_grad(); })) {
      auto mark = [&](const at::Tensor& t) {
        return (t.defined() ? t.detach() : at::empty({0}, grads[0].options())).requires_grad_(true);
      };
      const variable_list marked = NoThirdOrderRotary::apply(mark(d[0]), mark(d[1]), mark(d[2]), mark(d[3]), mark(d[4]), mark(d[5]));
      for (int i = 0; i < 6; ++i)
        if (d[i].defined()) d[i] = marked[i];
    }
    return {none, d[0], d[1], d[2], d[3], d[4], d[5], none, none, none, none};
  }
};

struct RotaryFn : public torch::autograd::Function<RotaryFn> {
  static variable_list forward(AutogradContext* ctx, const RotaryOptions& o, const at::Tensor& q, const at::Tensor& k,
                               const MaybeTensor& wq_, const MaybeTensor& wk_, const MaybeTensor& frequencies,
                               const MaybeTensor& positions, const MaybeTensor& lengths, const MaybeTensor& offsets) {
    const at::Tensor wq = given(wq_), wk = given(wk_);
    const RotaryWhere w{given(frequencies), given(positions), given(lengths), given(offsets)};
    auto [q_out, k_out] = rotary_fwd_core(q, k, wq, wk, w, o);
    RotarySaved::save(ctx, w, o, o.eps ? variable_list{q, k, wq, wk} : variable_list{});
    return {q_out, k_out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list r = ctx->get_saved_variables();
    const RotaryOptions o = RotarySaved::options(ctx);
    at::Tensor none;
    // (without norms the cotangents stand in for the rows, of which only the shapes matter)
    const at::Tensor q = o.eps ? r[4] : grads[0].detach(), k = o.eps ? r[5] : grads[1].detach();
    const at::Tensor wq = o.eps ? r[6] : none, wk = o.eps ? r[7] : none;
    if (!c10::GradMode::is_enabled()) {  // no graph, no node
      const auto [dq, dk, dwq, dwk] = rotary_bwd_core(q, k, wq, wk, grads[0], grads[1], RotarySaved::where(r), o);
      return {none, dq, dk, dwq, dwk, none, none, none, none};
    }
    const variable_list d = RotaryBwdFn::apply(o, q, k, maybe(wq), maybe(wk), grads[0], grads[1], maybe(r[0]), maybe(r[1]),
                                              maybe(r[2]), maybe(r[3]));
    return {none, d[0], d[1], wq.defined() ? d[2] : none, wk.defined() ? d[3] : none, none, none, none, none};
  }
};

// ----------------------------------------------------------- Python-facing

// Runs f without the GIL and raises its errors as Python exceptions.
template <class F>
auto py_call(F&& f) {
  try {
    py::gil_scoped_release nogil;
    return f();
  } catch (const ArgError& e) {
    throw py::value_error(e.what());
  } catch (const StatusError& e) {
    PyErr_SetObject(api().error_cls.ptr(), py::make_tuple(e.status, std::string(e.what())).ptr());
    throw py::error_already_set();
  }
}

std::tuple<at::Tensor, at::Tensor> attention_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                 int causal, double scale, int window, int sinks) {
  require_bound((const void*)api().fwd);
  return py_call([&] { return fwd_core(q, k, v, causal, scale, {window, sinks}); });
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> attention_bwd(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& o, const at::Tensor& dout,
    const at::Tensor& lse, int causal, double scale, int window, int sinks) {
  require_bound((const void*)api().bwd);
  return py_call([&] { return bwd_core(q, k, v, o, dout, lse, causal, scale, {window, sinks}); });
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> attention_bwdbwd(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& o, const at::Tensor& dout,
    const at::Tensor& ddq, const at::Tensor& ddk, const at::Tensor& ddv, const at::Tensor& lse, int causal,
    double scale, int window, int sinks) {
  require_bound((const void*)api().bwdbwd);
  return py_call([&] { return bwdbwd_core(q, k, v, o, dout, ddq, ddk, ddv, lse, causal, scale, {window, sinks}); });
}

at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                           const at::Tensor& table, const at::Tensor& lengths, const MaybeTensor& offsets,
                           const MaybeTensor& k_scale, const MaybeTensor& v_scale, int window, int sinks, double scale,
                           const MaybeTensor& out) {
  require_bound((const void*)api().paged_attention);
  return py_call([&] {
    return paged_attention_core(q, k_cache, v_cache, table, lengths, offsets, k_scale, v_scale, window, sinks, scale,
                                out);
  });
}

void paged_cache_write(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_cache, const at::Tensor& v_cache,
                       const at::Tensor& table, const at::Tensor& lengths, const MaybeTensor& offsets,
                       const MaybeTensor& k_scale, const MaybeTensor& v_scale) {
  require_bound((const void*)api().cache_write);
  py_call([&] { cache_write_core(k, v, k_cache, v_cache, table, lengths, offsets, k_scale, v_scale); });
}

std::tuple<at::Tensor, at::Tensor> paged_cache_read(const at::Tensor& k_cache, const at::Tensor& v_cache,
                                                    const at::Tensor& table, const at::Tensor& lengths,
                                                    int64_t max_length, at::ScalarType dtype,
                                                    const MaybeTensor& k_scale, const MaybeTensor& v_scale) {
  require_bound((const void*)api().cache_read);
  return py_call([&] { return cache_read_core(k_cache, v_cache, table, lengths, max_length, dtype, k_scale, v_scale); });
}

// O of attention(q, k, v) with the autograd nodes above (when q, k or v
// require grad and grad mode is on).
at::Tensor attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int64_t causal, double scale,
                     int64_t window, int64_t sinks) {
  require_bound((const void*)api().bwdbwd);
  return py_call([&] { return AttentionFn::apply(q, k, v, Mask{(int)causal, scale, {(int)window, (int)sinks}})[0]; });
}

at::Tensor paged_cache_extend(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& table,
                              const at::Tensor& lengths, const MaybeTensor& new_tokens, int new_each,
                              const MaybeTensor& parents, const MaybeTensor& k_scale, const MaybeTensor& v_scale) {
  require_bound((const void*)api().cache_extend);
  return py_call([&] {
    return cache_extend_core(k_cache, v_cache, table, lengths, new_tokens, new_each, parents, k_scale, v_scale);
  });
}

std::tuple<at::Tensor, at::Tensor, MaybeTensor, MaybeTensor, MaybeTensor, at::Tensor> paged_cache_compact(
    const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& table, const at::Tensor& lengths,
    int64_t num_pages, const MaybeTensor& k_scale, const MaybeTensor& v_scale, const MaybeTensor& key_means) {
  require_bound((const void*)api().cache_compact);
  return py_call([&] { return cache_compact_core(k_cache, v_cache, table, lengths, num_pages, k_scale, v_scale, key_means); });
}

void paged_key_means(const at::Tensor& k_cache, const at::Tensor& means, const at::Tensor& table,
                     const at::Tensor& lengths, const MaybeTensor& offsets, const MaybeTensor& k_scale) {
  require_bound((const void*)api().key_means);
  py_call([&] { key_means_core(k_cache, means, table, lengths, offsets, k_scale); });
}

at::Tensor paged_block_select(const at::Tensor& q, const at::Tensor& means, const at::Tensor& table,
                              const at::Tensor& lengths, const MaybeTensor& offsets, int64_t page_size, int64_t blocks,
                              int64_t first, int64_t last) {
  require_bound((const void*)api().block_select);
  return py_call([&] { return block_select_core(q, means, table, lengths, offsets, page_size, blocks, first, last); });
}

at::Tensor paged_block_attention(const at::Tensor& q, const at::Tensor& chosen, const at::Tensor& k_cache,
                                 const at::Tensor& v_cache, const at::Tensor& table, const at::Tensor& lengths,
                                 const MaybeTensor& offsets, const MaybeTensor& k_scale, const MaybeTensor& v_scale,
                                 double scale, const MaybeTensor& out) {
  require_bound((const void*)api().block_attention);
  return py_call([&] {
    return block_attention_core(q, chosen, k_cache, v_cache, table, lengths, offsets, k_scale, v_scale, scale, out);
  });
}

// qk_norm_rotary(q, k, ...) with the autograd nodes above (when q, k or a weight requires grad and grad mode is on);
// three axes: unbatched.
std::tuple<at::Tensor, at::Tensor> qk_norm_rotary(const at::Tensor& q, const at::Tensor& k, const MaybeTensor& wq,
                                                  const MaybeTensor& wk, const MaybeTensor& frequencies,
                                                  const MaybeTensor& positions, const MaybeTensor& lengths,
                                                  const MaybeTensor& offsets, bool interleaved,
                                                  c10::optional<double> eps) {
  require_bound((const void*)api().rotary_bwdbwd);
  return py_call([&]() -> std::tuple<at::Tensor, at::Tensor> {
    const at::Tensor a = given(wq), b = given(wk);
    const RotaryOptions o{interleaved, eps};
    if (c10::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || (a.defined() && a.requires_grad()) ||
                                        (b.defined() && b.requires_grad()))) {
      const variable_list out = RotaryFn::apply(o, q, k, wq, wk, frequencies, positions, lengths, offsets);
      return {out[0], out[1]};
    }
    return rotary_fwd_core(q, k, a, b, {given(frequencies), given(positions), given(lengths), given(offsets)}, o);
  });
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "Tensor-level calls of the Flash-HOG C ABI (see flash_hog/_hip.py)";
  m.def("bind", &bind, "bind(fwd, bwd, bwdbwd, last_error, status_string, error_cls): entry-point addresses");
  m.def("bind_window", &bind_window, "bind_window(workspace_bytes, fwd, bwd, bwdbwd): their addresses");
  m.def("bind_paged", &bind_paged, "bind_paged(workspace_bytes, attention, write, read): their addresses");
  m.def("bind_pages", &bind_pages, "bind_pages(workspace_bytes, extend, compact): their addresses");
  m.def("bind_blocks", &bind_blocks,
        "bind_blocks(key_means, select_workspace_bytes, select, workspace_bytes, attention): their addresses");
  m.def("bind_rotary", &bind_rotary, "bind_rotary(workspace_bytes, fwd, bwd, bwdbwd): their addresses");
  m.def("paged_cache_extend", &paged_cache_extend);
  m.def("paged_cache_compact", &paged_cache_compact);
  m.def("paged_key_means", &paged_key_means);
  m.def("paged_block_select", &paged_block_select);
  m.def("paged_block_attention", &paged_block_attention);
  m.def("qk_norm_rotary", &qk_norm_rotary);
  m.def("paged_attention", &paged_attention);
  m.def("paged_cache_write", &paged_cache_write);
  m.def("paged_cache_read", &paged_cache_read);
  using py::arg;
  m.def("attention_fwd", &attention_fwd, arg("q"), arg("k"), arg("v"), arg("causal"), arg("scale"), arg("window") = 0,
        arg("sinks") = 0);
  m.def("attention_bwd", &attention_bwd, arg("q"), arg("k"), arg("v"), arg("o"), arg("dout"), arg("lse"),
        arg("causal"), arg("scale"), arg("window") = 0, arg("sinks") = 0);
  m.def("attention_bwdbwd", &attention_bwdbwd, arg("q"), arg("k"), arg("v"), arg("o"), arg("dout"), arg("ddq"),
        arg("ddk"), arg("ddv"), arg("lse"), arg("causal"), arg("scale"), arg("window") = 0, arg("sinks") = 0);
  m.def("attention", &attention, "attention(q, k, v, causal, scale) -> O, differentiable twice", arg("q"), arg("k"),
        arg("v"), arg("causal"), arg("scale"), arg("window") = 0, arg("sinks") = 0);
}
