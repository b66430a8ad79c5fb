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
  const int* table_ptr() const { return table.data_ptr<int>(); }
  const int* lengths_ptr() const { return lengths.data_ptr<int>(); }
  const int* offsets_ptr() const { return offsets.defined() ? offsets.data_ptr<int>() : nullptr; }
};

// Tells autograd that a tensor was written to: a graph that saved it before then raises in its
// backward. (Inference tensors, which no graph can save, have no version.)
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Refuses an out whose memory a contiguous tensor that the kernels read shares; `same`: but for all
// of it, row by row.
void check_apart(const at::Tensor& out, const char* name, const at::Tensor& t, bool same) {
  const char *a = (const char*)out.data_ptr(), *b = (const char*)t.data_ptr();
  if (a < b + t.nbytes() && b < a + out.nbytes() && !(same && a == b))
    value_error(std::string("out overlaps ") + name);
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
    check_apart(out, "query", q, true);
    check_apart(out, "key_cache", k_cache, false);
    check_apart(out, "value_cache", v_cache, false);
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

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "Tensor-level calls of the Flash-HOG C ABI (see flash_hog/_hip.py)";
  m.def("bind", &bind, "bind(fwd, bwd, bwdbwd, last_error, status_string, error_cls): entry-point addresses");
  m.def("bind_window", &bind_window, "bind_window(workspace_bytes, fwd, bwd, bwdbwd): their addresses");
  m.def("bind_paged", &bind_paged, "bind_paged(workspace_bytes, attention, write, read): their addresses");
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
