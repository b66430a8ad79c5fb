"""ctypes binding of libflash_hog_hip.so, the C ABI declared in include/flash_hog.h.

This mirrors the plugin loader of the reference's native path
(flash_hog/jax/_tk_gpu.py:26-58): the library path comes from the
FLASH_HOG_HIP_LIB environment variable or the in-tree build, the library is
loaded once, and a missing library is an error (there is no fallback path).

The torch-level helpers below take device tensors, check them, allocate the
outputs and the fp32 row-statistic workspace with torch's caching allocator,
and enqueue the kernels on torch's current stream for the tensors' device.
Their `causal` argument is a bool (top-left when true) or the C ABI's code
(0 none, 1 top-left, 2 bottom-right). attention_fwd, attention_bwd and
attention_bwdbwd hand the work to the torch extension _lib/_fhog_torch when
it is built (the same checks, allocations and C-ABI call in C++, a few
microseconds of host time instead of 9-20), bound to the entry points of the
library loaded here; FLASH_HOG_TORCH_EXT=0 keeps them in Python.
"""

from __future__ import annotations

import ctypes
import functools
import importlib.machinery
import importlib.util
import os
import pathlib
import sysconfig
import warnings

import torch

LIB_ENV = "FLASH_HOG_HIP_LIB"
LIB_PATH = pathlib.Path(__file__).resolve().parent / "_lib" / "libflash_hog_hip.so"

FHOG_OK = 0
FHOG_ERR_INVALID_ARGUMENT = 1
FHOG_ERR_UNSUPPORTED = 2
FHOG_ERR_LAUNCH = 3

DTYPE_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}

_p = ctypes.c_void_p
_i = ctypes.c_int
_f = ctypes.c_float

SIGNATURES = {
    "fhog_abi_version": (_i, []),
    "fhog_status_string": (ctypes.c_char_p, [_i]),
    "fhog_last_error": (ctypes.c_char_p, []),
    "fhog_row_stat_bytes": (ctypes.c_size_t, [_i, _i, _i]),
    "fhog_attention_supported": (_i, [_i] * 9 + [_f]),
    "fhog_attention_fwd": (_i, [_p, _p, _p, _p, _p, _p] + [_i] * 8 + [_f]),
    "fhog_attention_bwd": (_i, [_p] * 11 + [_i] * 8 + [_f]),
    "fhog_attention_bwdbwd": (_i, [_p] * 17 + [_i] * 8 + [_f]),
    "fhog_attention_bwdbwd_stage": (_i, [_p, _i] + [_p] * 16 + [_i] * 8 + [_f]),
    "fhog_attention_bwdbwd_noalloc": (_i, [_p] * 14 + [_i] * 8 + [_f]),
    "fhog_window_workspace_bytes": (ctypes.c_size_t, [_i] * 10),
    "fhog_window_attention_fwd": (_i, [_p] * 6 + [_i] * 10 + [_f]),
    "fhog_window_attention_bwd": (_i, [_p] * 12 + [_i] * 10 + [_f]),
    "fhog_window_attention_bwdbwd": (_i, [_p] * 18 + [_i] * 10 + [_f]),
    "fhog_paged_workspace_bytes": (ctypes.c_size_t, [_i] * 10),
    "fhog_paged_attention": (_i, [_p] * 11 + [ctypes.c_size_t] + [_i] * 13 + [_f]),
    "fhog_paged_cache_write": (_i, [_p] * 10 + [_i] * 9),
    "fhog_paged_cache_read": (_i, [_p] * 9 + [_i] * 9),
    "fhog_paged_pages_workspace_bytes": (ctypes.c_size_t, [_i] * 3),
    "fhog_paged_cache_extend": (_i, [_p] * 9 + [_i, _p, _p, ctypes.c_size_t] + [_i] * 7),
    "fhog_paged_cache_compact": (_i, [_p] * 15 + [ctypes.c_size_t] + [_i] * 8),
    "fhog_paged_key_means": (_i, [_p] * 7 + [_i] * 7),
    "fhog_paged_block_select_workspace_bytes": (ctypes.c_size_t, [_i] * 8),
    "fhog_paged_block_select": (_i, [_p] * 8 + [ctypes.c_size_t] + [_i] * 12),
    "fhog_paged_block_workspace_bytes": (ctypes.c_size_t, [_i] * 9),
    "fhog_paged_block_attention": (_i, [_p] * 12 + [ctypes.c_size_t] + [_i] * 12 + [_f]),
    "fhog_qk_norm_rotary_workspace_bytes": (ctypes.c_size_t, [_p]),
    "fhog_qk_norm_rotary_fwd": (_i, [_p] * 8),
    "fhog_qk_norm_rotary_bwd": (_i, [_p] * 13),
    "fhog_qk_norm_rotary_bwdbwd": (_i, [_p] * 19),
}


class Rotary(ctypes.Structure):
    """fhog_rotary."""

    _fields_ = ([(n, _i) for n in ("batch", "tokens", "heads", "kv_heads", "head_dim", "rotated", "dtype",
                                   "weight_dtype", "interleaved", "norm")]
                + [("eps", _f)] + [(n, _i) for n in ("position_bytes", "position_rows", "sequences")]
                + [(n, ctypes.c_longlong * 3) for n in ("q_stride", "k_stride")]
                + [(n, _p) for n in ("frequencies", "positions", "lengths", "query_offsets")])


class FlashHogError(RuntimeError):
    """A C-ABI call returned a non-zero status."""

    def __init__(self, status: int, message: str):
        super().__init__(message)
        self.status = status


def library_path() -> pathlib.Path:
    return pathlib.Path(os.environ.get(LIB_ENV) or LIB_PATH)


@functools.cache
def lib() -> ctypes.CDLL:
    path = library_path()
    if not path.exists():
        raise ImportError(
            f"Flash-HOG HIP library not found at {path}; build it with "
            f"`python flash-hog_amd/build.py` (or set {LIB_ENV})")
    handle = ctypes.CDLL(str(path))
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(handle, name)
        fn.restype = res
        fn.argtypes = args
    return handle


TORCH_EXT_ENV = "FLASH_HOG_TORCH_EXT"
TORCH_EXT_PATH = LIB_PATH.parent / ("_fhog_torch" + sysconfig.get_config_var("EXT_SUFFIX"))


@functools.cache
def torch_ext():
    """The _fhog_torch extension bound to lib()'s entry points, or None when it
    is not built, cannot be loaded (built for another torch or Python, an
    undefined symbol: a warning says why, once) or FLASH_HOG_TORCH_EXT=0; the
    Python wrappers then do the same work. A missing kernel library is still
    an error (lib() raises), since the wrappers need it too. The result,
    None included, is cached."""
    if os.environ.get(TORCH_EXT_ENV, "1") == "0" or not TORCH_EXT_PATH.exists():
        return None
    L = lib()
    name = "flash_hog._lib._fhog_torch"
    try:
        loader = importlib.machinery.ExtensionFileLoader(name, str(TORCH_EXT_PATH))
        mod = importlib.util.module_from_spec(importlib.util.spec_from_loader(name, loader))
        loader.exec_module(mod)
        addr = lambda fn: ctypes.cast(fn, ctypes.c_void_p).value
        mod.bind(addr(L.fhog_attention_fwd), addr(L.fhog_attention_bwd), addr(L.fhog_attention_bwdbwd),
                 addr(L.fhog_last_error), addr(L.fhog_status_string), FlashHogError)
        mod.bind_window(addr(L.fhog_window_workspace_bytes), addr(L.fhog_window_attention_fwd),
                        addr(L.fhog_window_attention_bwd), addr(L.fhog_window_attention_bwdbwd))
        mod.bind_paged(addr(L.fhog_paged_workspace_bytes), addr(L.fhog_paged_attention),
                       addr(L.fhog_paged_cache_write), addr(L.fhog_paged_cache_read))
        mod.bind_pages(addr(L.fhog_paged_pages_workspace_bytes), addr(L.fhog_paged_cache_extend),
                       addr(L.fhog_paged_cache_compact))
        mod.bind_blocks(addr(L.fhog_paged_key_means), addr(L.fhog_paged_block_select_workspace_bytes),
                        addr(L.fhog_paged_block_select), addr(L.fhog_paged_block_workspace_bytes),
                        addr(L.fhog_paged_block_attention))
        mod.bind_rotary(addr(L.fhog_qk_norm_rotary_workspace_bytes), addr(L.fhog_qk_norm_rotary_fwd),
                        addr(L.fhog_qk_norm_rotary_bwd), addr(L.fhog_qk_norm_rotary_bwdbwd))
    except (ImportError, OSError, AttributeError) as exc:
        warnings.warn(f"Flash-HOG torch extension {TORCH_EXT_PATH} not loaded ({exc}); "
                      "using the Python wrappers", RuntimeWarning, stacklevel=2)
        return None
    return mod


def check(status: int) -> None:
    if status != FHOG_OK:
        L = lib()
        msg = L.fhog_last_error().decode() or L.fhog_status_string(status).decode()
        raise FlashHogError(status, msg)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


class _on_device:
    """Makes `device` current for the duration of a kernel call (the C ABI
    enqueues on the stream it is given, but the launch runs on the current
    device); a no-op when it already is."""

    __slots__ = ("index", "prev")

    def __init__(self, device: torch.device):
        self.index = device.index

    def __enter__(self):
        self.prev = torch.cuda.current_device()
        if self.prev != self.index:
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.prev != self.index:
            torch.cuda.set_device(self.prev)
        return False


def _check_inputs(named, dtype=None):
    first = None
    for name, t in named:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if not t.is_cuda:
            raise ValueError(f"{name} must be on a GPU device, got {t.device}")
        if first is None:
            first = t
            dev = t.get_device()
        elif t.get_device() != dev:
            raise ValueError(f"{name} is on {t.device}, expected {first.device}")
        if dtype is not None and t.dtype != dtype:
            raise ValueError(f"{name} has dtype {t.dtype}, expected {dtype}")
    return first


def _contig(*xs):
    return tuple(x if x.is_contiguous() else x.contiguous() for x in xs)


def _dims(q: torch.Tensor, k: torch.Tensor):
    """(B, Tq, Tk, N, Nk, H) of q (B, Tq, N, H) and k (B, Tk, Nk, H); N must be a
    multiple of Nk (grouped-query attention when N > Nk)."""
    if q.ndim != 4 or k.ndim != 4:
        raise ValueError(f"expected (B, T, N, H) tensors, got q{tuple(q.shape)} k{tuple(k.shape)}")
    B, Tq, N, Hd = q.shape
    Bk, Tk, Nk, Hk = k.shape
    if Bk != B or Hk != Hd:
        raise ValueError(f"q{tuple(q.shape)} and k{tuple(k.shape)} disagree on batch or head_dim")
    if Nk == 0 or N % Nk != 0:
        raise ValueError(f"query heads ({N}) must be a multiple of key/value heads ({Nk})")
    if q.dtype not in DTYPE_CODES:
        raise ValueError(f"unsupported dtype {q.dtype}")
    return B, Tq, Tk, N, Nk, Hd


def causal_code(causal) -> int:
    """C ABI causal code: False/True map to none/top-left; ints pass through
    (0 none, 1 top-left, 2 bottom-right; the library rejects others)."""
    return int(causal)


def _expect(name, t, shape, dtype=None):
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} has dtype {t.dtype}, expected {dtype}")


def attention_supported(batch: int, n_q: int, n_k: int, heads: int, kv_heads: int, head_dim: int, dtype,
                        causal, scale: float, device: int = -1) -> tuple[bool, str]:
    """(True, "") if the library has kernels for these arguments (and, for
    device >= 0, that HIP device is a gfx950 GPU), else (False, the reason the
    entry points would give). Launches and allocates nothing."""
    if dtype not in DTYPE_CODES:
        return False, f"unsupported dtype {dtype}"
    status = lib().fhog_attention_supported(int(device), batch, n_q, n_k, heads, kv_heads, head_dim,
                                            DTYPE_CODES[dtype], causal_code(causal), float(scale))
    return status == 0, "" if status == 0 else lib().fhog_last_error().decode()


def _window_args(window: int, sinks: int):
    """window and sinks as the C ABI's ints; window 0 is none."""
    window, sinks = int(window), int(sinks)
    if window < 0 or sinks < 0 or (sinks and not window):
        raise ValueError(f"window must be >= 1 (or 0: none) and sinks >= 0 (0 without a window), got {window}, {sinks}")
    return min(window, (1 << 31) - 1), min(sinks, (1 << 31) - 1)


def _window_workspace(q, dims, causal, window, sinks):
    """Workspace of a windowed backward (fhog_window_workspace_bytes), or None where it needs none."""
    size = lib().fhog_window_workspace_bytes(*dims, DTYPE_CODES[q.dtype], causal_code(causal), window, sinks)
    return torch.empty(size, device=q.device, dtype=torch.uint8) if size else None


def attention_fwd(q, k, v, causal, scale: float, window: int = 0, sinks: int = 0):
    """O (B, T, N, H) in q's dtype and the natural-log logsumexp L (B, N, T) fp32.
    window > 0 (here and below; causal masks only): the last `window` keys up to a
    query's own position and the first `sinks` keys are visible to it."""
    window, sinks = _window_args(window, sinks)
    ext = torch_ext()
    if ext is not None:
        return ext.attention_fwd(q, k, v, causal_code(causal), float(scale), window, sinks)
    _check_inputs([("q", q), ("k", k), ("v", v)], q.dtype)
    B, Tq, Tk, N, Nk, Hd = _dims(q, k)
    _expect("v", v, k.shape)
    q, k, v = _contig(q, k, v)
    o = torch.empty_like(q)
    lse = torch.empty((B, N, Tq), device=q.device, dtype=torch.float32)
    with _on_device(q.device):
        args = (_stream(q.device), _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(lse),
                B, Tq, Tk, N, Nk, Hd, DTYPE_CODES[q.dtype], causal_code(causal))
        if window:
            check(lib().fhog_window_attention_fwd(*args, window, sinks, float(scale)))
        else:
            check(lib().fhog_attention_fwd(*args, float(scale)))
    return o, lse


def attention_bwd(q, k, v, o, dout, lse, causal, scale: float, window: int = 0, sinks: int = 0):
    """dQ, dK, dV of attention given its residual; also returns D (B, N, T) fp32."""
    window, sinks = _window_args(window, sinks)
    ext = torch_ext()
    if ext is not None:
        return ext.attention_bwd(q, k, v, o, dout, lse, causal_code(causal), float(scale), window, sinks)
    _check_inputs([("q", q), ("k", k), ("v", v), ("o", o), ("dout", dout)], q.dtype)
    _check_inputs([("q", q), ("lse", lse)])
    B, Tq, Tk, N, Nk, Hd = _dims(q, k)
    _expect("v", v, k.shape)
    _expect("o", o, q.shape)
    _expect("dout", dout, q.shape)
    _expect("lse", lse, (B, N, Tq), torch.float32)
    q, k, v, o, dout, lse = _contig(q, k, v, o, dout, lse)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    delta = torch.empty((B, N, Tq), device=q.device, dtype=torch.float32)
    with _on_device(q.device):
        ptrs = (_stream(q.device), _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(dout), _ptr(lse),
                _ptr(dq), _ptr(dk), _ptr(dv), _ptr(delta))
        sizes = (B, Tq, Tk, N, Nk, Hd, DTYPE_CODES[q.dtype], causal_code(causal))
        if window:
            ws = _window_workspace(q, (B, Tq, Tk, N, Nk, Hd), causal, window, sinks)
            check(lib().fhog_window_attention_bwd(*ptrs, _ptr(ws), *sizes, window, sinks, float(scale)))
        else:
            check(lib().fhog_attention_bwd(*ptrs, *sizes, float(scale)))
    return dq, dk, dv, delta


def attention_bwdbwd(q, k, v, o, dout, ddq, ddk, ddv, lse, causal, scale: float,
                     return_stats: bool = False, window: int = 0, sinks: int = 0):
    """dQ2, dK2, dV2, ddO of the double backward [and the row statistics D, dD, B]."""
    window, sinks = _window_args(window, sinks)
    ext = torch_ext()
    if ext is not None:
        dq2, dk2, dv2, ddo, stats = ext.attention_bwdbwd(q, k, v, o, dout, ddq, ddk, ddv, lse, causal_code(causal),
                                                         float(scale), window, sinks)
        return (dq2, dk2, dv2, ddo, tuple(stats.unbind(0))) if return_stats else (dq2, dk2, dv2, ddo)
    _check_inputs([("q", q), ("k", k), ("v", v), ("o", o), ("dout", dout),
                   ("ddq", ddq), ("ddk", ddk), ("ddv", ddv)], q.dtype)
    _check_inputs([("q", q), ("lse", lse)])
    B, Tq, Tk, N, Nk, Hd = _dims(q, k)
    _expect("v", v, k.shape)
    for name, t in (("o", o), ("dout", dout), ("ddq", ddq)):
        _expect(name, t, q.shape)
    for name, t in (("ddk", ddk), ("ddv", ddv)):
        _expect(name, t, k.shape)
    _expect("lse", lse, (B, N, Tq), torch.float32)
    q, k, v, o, dout, ddq, ddk, ddv, lse = _contig(q, k, v, o, dout, ddq, ddk, ddv, lse)
    dq2, dk2, dv2, ddo = (torch.empty_like(x) for x in (q, k, v, dout))
    stats = torch.empty((3, B, N, Tq), device=q.device, dtype=torch.float32)
    with _on_device(q.device):
        ptrs = (_stream(q.device), _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(dout),
                _ptr(ddq), _ptr(ddk), _ptr(ddv), _ptr(lse),
                _ptr(dq2), _ptr(dk2), _ptr(dv2), _ptr(ddo),
                _ptr(stats[0]), _ptr(stats[1]), _ptr(stats[2]))
        sizes = (B, Tq, Tk, N, Nk, Hd, DTYPE_CODES[q.dtype], causal_code(causal))
        if window:
            ws = _window_workspace(q, (B, Tq, Tk, N, Nk, Hd), causal, window, sinks)
            check(lib().fhog_window_attention_bwdbwd(*ptrs, _ptr(ws), *sizes, window, sinks, float(scale)))
        else:
            check(lib().fhog_attention_bwdbwd(*ptrs, *sizes, float(scale)))
    if return_stats:
        return dq2, dk2, dv2, ddo, (stats[0], stats[1], stats[2])
    return dq2, dk2, dv2, ddo


def attention_bwdbwd_noalloc(q, k, v, o, dout, ddq, ddk, ddv, lse, causal, scale: float, out=None):
    """attention_bwdbwd through fhog_attention_bwdbwd_noalloc: the row
    statistics live in the library's static device scratch, so the call needs
    no workspace. `out` = (dq2, dk2, dv2, ddo) preallocated outputs (allocated
    here when None)."""
    _check_inputs([("q", q), ("k", k), ("v", v), ("o", o), ("dout", dout),
                   ("ddq", ddq), ("ddk", ddk), ("ddv", ddv)], q.dtype)
    _check_inputs([("q", q), ("lse", lse)])
    B, Tq, Tk, N, Nk, Hd = _dims(q, k)
    _expect("v", v, k.shape)
    for name, t in (("o", o), ("dout", dout), ("ddq", ddq)):
        _expect(name, t, q.shape)
    for name, t in (("ddk", ddk), ("ddv", ddv)):
        _expect(name, t, k.shape)
    _expect("lse", lse, (B, N, Tq), torch.float32)
    q, k, v, o, dout, ddq, ddk, ddv, lse = _contig(q, k, v, o, dout, ddq, ddk, ddv, lse)
    if out is None:
        out = tuple(torch.empty_like(x) for x in (q, k, v, dout))
    for name, t, like in zip(("dq2", "dk2", "dv2", "ddo"), out, (q, k, v, dout)):
        _expect(name, t, like.shape, like.dtype)
        if not t.is_contiguous() or t.device != q.device:
            raise ValueError(f"{name} must be contiguous on {q.device}")
    dq2, dk2, dv2, ddo = out
    with _on_device(q.device):
        check(lib().fhog_attention_bwdbwd_noalloc(
            _stream(q.device), _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(dout),
            _ptr(ddq), _ptr(ddk), _ptr(ddv), _ptr(lse),
            _ptr(dq2), _ptr(dk2), _ptr(dv2), _ptr(ddo),
            B, Tq, Tk, N, Nk, Hd, DTYPE_CODES[q.dtype], causal_code(causal), float(scale)))
    return dq2, dk2, dv2, ddo


# ------------------------------------------------------------- paged cache

CACHE_DTYPE_CODES = {**DTYPE_CODES, torch.float8_e4m3fn: 3}  # (the library refuses an fp32 one)
_SCALE_DTYPES = (torch.float8_e8m0fnu, torch.uint8)


def _check_cache(first, k_cache, v_cache, page_table, lengths, query_offsets, k_scale, v_scale, dtype):
    """Checks a paged cache and what finds tokens in it; `first` is the (name, tensor) whose
    device all share. Returns (num_pages, kv_heads, page_size, head_dim, batch, pages_per_seq)
    and the index tensors, contiguous."""
    named = [first, ("key_cache", k_cache), ("value_cache", v_cache), ("page_table", page_table),
             ("lengths", lengths)]
    quantised = k_cache.dtype == torch.float8_e4m3fn
    if quantised:
        if k_scale is None or v_scale is None:
            raise ValueError("an e4m3 cache needs key_scale and value_scale")
        named += [("key_scale", k_scale), ("value_scale", v_scale)]
    elif k_scale is not None or v_scale is not None:
        raise ValueError(f"key_scale and value_scale are for an e4m3 cache, not {k_cache.dtype}")
    if query_offsets is not None:
        named.append(("query_offsets", query_offsets))
    _check_inputs(named)
    if k_cache.ndim != 4:
        raise ValueError(f"expected a (pages, kv_heads, page_size, head_dim) cache, got {tuple(k_cache.shape)}")
    _expect("value_cache", v_cache, k_cache.shape, k_cache.dtype)
    if k_cache.dtype not in (dtype, torch.float8_e4m3fn):
        raise ValueError(f"the cache must be of {dtype} or torch.float8_e4m3fn, got {k_cache.dtype}")
    for name, t in (("key_cache", k_cache), ("value_cache", v_cache)):
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    if quantised:
        for name, t in (("key_scale", k_scale), ("value_scale", v_scale)):
            _expect(name, t, k_cache.shape[:3])
            if t.dtype not in _SCALE_DTYPES or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous tensor of torch.float8_e8m0fnu or torch.uint8")
    if page_table.ndim != 2:
        raise ValueError(f"expected a (batch, pages) page_table, got {tuple(page_table.shape)}")
    batch = page_table.shape[0]
    _expect("lengths", lengths, (batch,))
    index = [("page_table", page_table), ("lengths", lengths)]
    if query_offsets is not None:
        _expect("query_offsets", query_offsets, (batch + 1,))
        index.append(("query_offsets", query_offsets))
    for name, t in index:
        if t.dtype != torch.int32:
            raise ValueError(f"{name} has dtype {t.dtype}, expected torch.int32")
    page_table, lengths = _contig(page_table, lengths)
    if query_offsets is not None:
        query_offsets = query_offsets.contiguous()
    return (*k_cache.shape, batch, page_table.shape[1]), page_table, lengths, query_offsets


def _overlap(a, b) -> bool:
    return a.data_ptr() < b.data_ptr() + b.nbytes and b.data_ptr() < a.data_ptr() + a.nbytes


def _check_apart(out, name, t, same=False):
    """Refuses an out whose memory a contiguous tensor that the kernels read shares; same: but for all
    of it, row by row."""
    if _overlap(out, t) and not (same and out.data_ptr() == t.data_ptr()):
        raise ValueError(f"out overlaps {name}")


def _check_apart_from(out_name, out, k_cache, v_cache, k_scale, v_scale, page_table, lengths, query_offsets):
    """Refuses an out that shares memory with a cache or with what finds tokens in it."""
    for name, t in (("key_cache", k_cache), ("value_cache", v_cache), ("key_scale", k_scale), ("value_scale", v_scale),
                    ("page_table", page_table), ("lengths", lengths), ("query_offsets", query_offsets)):
        if t is not None and _overlap(out, t):
            raise ValueError(f"{out_name} overlaps {name}")


def _written(*tensors):
    """Tells autograd that tensors were written to: a graph that saved one before then raises in its
    backward. (Inference tensors, which no graph can save, have no version.)"""
    torch.autograd.graph.increment_version([t for t in tensors if t is not None and not t.is_inference()])


def paged_attention(q, k_cache, v_cache, page_table, lengths, query_offsets, k_scale, v_scale, window: int,
                    sinks: int, scale: float, out=None):
    """out (T, N, H) of the packed new tokens q over a paged cache (fhog_paged_attention); window 0: none."""
    window, sinks = _window_args(window, sinks)
    ext = torch_ext()
    if ext is not None:
        return ext.paged_attention(q, k_cache, v_cache, page_table, lengths, query_offsets, k_scale, v_scale, window,
                                   sinks, float(scale), out)
    if q.ndim != 3:
        raise ValueError(f"expected a (T, N, H) query, got {tuple(q.shape)}")
    (pages, Nk, page, Hd, B, width), page_table, lengths, query_offsets = _check_cache(
        ("query", q), k_cache, v_cache, page_table, lengths, query_offsets, k_scale, v_scale, q.dtype)
    T, N, Hq = q.shape
    if Hq != Hd:
        raise ValueError(f"query{tuple(q.shape)} and key_cache{tuple(k_cache.shape)} disagree on head_dim")
    if q.dtype not in DTYPE_CODES:
        raise ValueError(f"unsupported dtype {q.dtype}")
    clear = out is None
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _check_inputs([("query", q), ("out", out)], q.dtype)
        _expect("out", out, q.shape)
        if not out.is_contiguous():
            raise ValueError("out must be contiguous")
    q = q.contiguous()
    if not clear:
        _check_apart(out, "query", q, same=True)
        _check_apart_from("out", out, k_cache, v_cache, k_scale, v_scale, page_table, lengths, query_offsets)
    with _on_device(q.device):
        size = lib().fhog_paged_workspace_bytes(B, T, int(query_offsets is None), N, Nk, Hd, page, width, window, sinks)
        ws = torch.empty(size, device=q.device, dtype=torch.uint8) if size else None
        check(lib().fhog_paged_attention(
            _stream(q.device), _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale), _ptr(page_table),
            _ptr(lengths), _ptr(query_offsets), _ptr(out), _ptr(ws), size, B, T, N, Nk, Hd, pages, page, width,
            DTYPE_CODES[q.dtype], CACHE_DTYPE_CODES[k_cache.dtype], window, sinks, int(clear), float(scale)))
    if not clear:
        _written(out)
    return out


def paged_cache_write(k, v, k_cache, v_cache, page_table, lengths, query_offsets, k_scale, v_scale) -> None:
    """The packed new tokens' keys and values (T, N, H) into their pages (fhog_paged_cache_write)."""
    ext = torch_ext()
    if ext is not None:
        ext.paged_cache_write(k, v, k_cache, v_cache, page_table, lengths, query_offsets, k_scale, v_scale)
        return
    if k.ndim != 3:
        raise ValueError(f"expected a (T, N, H) key, got {tuple(k.shape)}")
    (pages, Nk, page, Hd, B, width), page_table, lengths, query_offsets = _check_cache(
        ("key", k), k_cache, v_cache, page_table, lengths, query_offsets, k_scale, v_scale, k.dtype)
    _check_inputs([("key", k), ("value", v)], k.dtype)
    _expect("value", v, k.shape)
    if tuple(k.shape[1:]) != (Nk, Hd):
        raise ValueError(f"key{tuple(k.shape)} and key_cache{tuple(k_cache.shape)} disagree on heads or head_dim")
    if k.dtype not in DTYPE_CODES:
        raise ValueError(f"unsupported dtype {k.dtype}")
    k, v = _contig(k, v)
    with _on_device(k.device):
        check(lib().fhog_paged_cache_write(
            _stream(k.device), _ptr(k), _ptr(v), _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale),
            _ptr(page_table), _ptr(lengths), _ptr(query_offsets), B, k.shape[0], Nk, Hd, pages, page, width,
            DTYPE_CODES[k.dtype], CACHE_DTYPE_CODES[k_cache.dtype]))
    _written(k_cache, v_cache, k_scale, v_scale)


def paged_cache_read(k_cache, v_cache, page_table, lengths, max_length: int, dtype, k_scale, v_scale):
    """The sequences' keys and values (B, max_length, N, H) in dtype, zeros behind their lengths
    (fhog_paged_cache_read)."""
    ext = torch_ext()
    if ext is not None:
        return ext.paged_cache_read(k_cache, v_cache, page_table, lengths, max_length, dtype, k_scale, v_scale)
    (pages, Nk, page, Hd, B, width), page_table, lengths, _ = _check_cache(
        ("key_cache", k_cache), k_cache, v_cache, page_table, lengths, None, k_scale, v_scale, dtype)
    if max_length < 0:
        raise ValueError(f"max_length must be >= 0, got {max_length}")
    if dtype not in DTYPE_CODES:
        raise ValueError(f"unsupported dtype {dtype}")
    k, v = (torch.empty((B, max_length, Nk, Hd), device=k_cache.device, dtype=dtype) for _ in range(2))
    with _on_device(k_cache.device):
        check(lib().fhog_paged_cache_read(
            _stream(k_cache.device), _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale), _ptr(page_table),
            _ptr(lengths), _ptr(k), _ptr(v), B, max_length, Nk, Hd, pages, page, width, DTYPE_CODES[dtype],
            CACHE_DTYPE_CODES[k_cache.dtype]))
    return k, v


def paged_cache_extend(k_cache, v_cache, page_table, lengths, new_tokens, new_each: int, parents, k_scale, v_scale):
    """Rows of page_table and lengths go on from their parents and grow by new_tokens (None: new_each) tokens,
    in place (fhog_paged_cache_extend); returns the free pages left, an int32 tensor of no axes."""
    ext = torch_ext()
    if ext is not None:
        return ext.paged_cache_extend(k_cache, v_cache, page_table, lengths, new_tokens, new_each, parents, k_scale,
                                      v_scale)
    (pages, Nk, page, Hd, B, width), _, _, _ = _check_cache(
        ("key_cache", k_cache), k_cache, v_cache, page_table, lengths, None, k_scale, v_scale, k_cache.dtype)
    if k_cache.dtype not in CACHE_DTYPE_CODES:
        raise ValueError(f"unsupported dtype {k_cache.dtype}")
    for name, t in (("page_table", page_table), ("lengths", lengths)):
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    for name, t in (("parents", parents), ("new_tokens", new_tokens)):
        if t is None:
            continue
        _check_inputs([("key_cache", k_cache), (name, t)])
        _expect(name, t, (B,), torch.int32)
        if _overlap(t, page_table) or _overlap(t, lengths):
            raise ValueError(f"{name} overlaps page_table or lengths")
    if B == 0:
        raise ValueError("expected at least one row of page_table")
    parents, new_tokens = (None if t is None else t.contiguous() for t in (parents, new_tokens))
    free = torch.empty((), device=k_cache.device, dtype=torch.int32)
    with _on_device(k_cache.device):
        size = lib().fhog_paged_pages_workspace_bytes(B, pages, width)
        ws = torch.empty(size, device=k_cache.device, dtype=torch.uint8)
        check(lib().fhog_paged_cache_extend(
            _stream(k_cache.device), _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale), _ptr(page_table),
            _ptr(lengths), _ptr(parents), _ptr(new_tokens), new_each, _ptr(free), _ptr(ws), size, B, Nk, Hd, pages, page,
            width, CACHE_DTYPE_CODES[k_cache.dtype]))
    _written(k_cache, v_cache, k_scale, v_scale, page_table, lengths)
    return free


def paged_cache_compact(k_cache, v_cache, page_table, lengths, num_pages: int, k_scale, v_scale, key_means):
    """(k_cache, v_cache, k_scale, v_scale, key_means, page_table): the used pages as the first of new caches
    of num_pages pages (fhog_paged_cache_compact); None for what is not given."""
    ext = torch_ext()
    if ext is not None:
        return ext.paged_cache_compact(k_cache, v_cache, page_table, lengths, num_pages, k_scale, v_scale, key_means)
    (pages, Nk, page, Hd, B, width), page_table, lengths, _ = _check_cache(
        ("key_cache", k_cache), k_cache, v_cache, page_table, lengths, None, k_scale, v_scale, k_cache.dtype)
    if k_cache.dtype not in CACHE_DTYPE_CODES:
        raise ValueError(f"unsupported dtype {k_cache.dtype}")
    if key_means is not None:
        _check_key_means(key_means, ("key_cache", k_cache), (pages, Nk, Hd))
    if num_pages < 1 or num_pages > (1 << 31) - 1:
        raise ValueError(f"num_pages must be >= 1 and below 2 ** 31, got {num_pages}")
    inputs = (k_cache, v_cache, k_scale, v_scale, key_means)
    outs = tuple(None if t is None else torch.empty((num_pages, *t.shape[1:]), device=t.device, dtype=t.dtype)
                 for t in inputs)
    table = torch.empty_like(page_table)
    with _on_device(k_cache.device):
        size = lib().fhog_paged_pages_workspace_bytes(B, pages, width)
        ws = torch.empty(size, device=k_cache.device, dtype=torch.uint8)
        check(lib().fhog_paged_cache_compact(
            _stream(k_cache.device), *map(_ptr, inputs), _ptr(page_table), _ptr(lengths), *map(_ptr, outs), _ptr(table),
            _ptr(ws), size, B, Nk, Hd, pages, page, width, num_pages, CACHE_DTYPE_CODES[k_cache.dtype]))
    return (*outs, table)


def _check_key_means(means, first, shape):
    _check_inputs([first, ("key_means", means)])
    _expect("key_means", means, shape, torch.float32)
    if not means.is_contiguous():
        raise ValueError("key_means must be contiguous")


def _check_index(first, page_table, lengths, query_offsets):
    """_check_cache's checks of what finds tokens; the contiguous tensors."""
    named = [("page_table", page_table), ("lengths", lengths)]
    if query_offsets is not None:
        named.append(("query_offsets", query_offsets))
    _check_inputs([first, *named])
    if page_table.ndim != 2:
        raise ValueError(f"expected a (batch, pages) page_table, got {tuple(page_table.shape)}")
    _expect("lengths", lengths, (page_table.shape[0],))
    if query_offsets is not None:
        _expect("query_offsets", query_offsets, (page_table.shape[0] + 1,))
    for name, t in named:
        if t.dtype != torch.int32:
            raise ValueError(f"{name} has dtype {t.dtype}, expected torch.int32")
    return tuple(None if t is None else t.contiguous() for t in (page_table, lengths, query_offsets))


def paged_key_means(k_cache, key_means, page_table, lengths, query_offsets, k_scale) -> None:
    """The means of the pages that the new tokens fill, into key_means (fhog_paged_key_means)."""
    ext = torch_ext()
    if ext is not None:
        ext.paged_key_means(k_cache, key_means, page_table, lengths, query_offsets, k_scale)
        return
    (pages, Nk, page, Hd, B, width), page_table, lengths, query_offsets = _check_cache(
        ("key_cache", k_cache), k_cache, k_cache, page_table, lengths, query_offsets, k_scale, k_scale, k_cache.dtype)
    if k_cache.dtype not in CACHE_DTYPE_CODES:
        raise ValueError(f"unsupported dtype {k_cache.dtype}")
    _check_key_means(key_means, ("key_cache", k_cache), (pages, Nk, Hd))
    _check_apart_from("key_means", key_means, k_cache, None, k_scale, None, page_table, lengths, query_offsets)
    with _on_device(k_cache.device):
        check(lib().fhog_paged_key_means(
            _stream(k_cache.device), _ptr(k_cache), _ptr(k_scale), _ptr(key_means), _ptr(page_table), _ptr(lengths),
            _ptr(query_offsets), B, Nk, Hd, pages, page, width, CACHE_DTYPE_CODES[k_cache.dtype]))
    _written(key_means)


def paged_block_select(q, key_means, page_table, lengths, query_offsets, page_size: int, blocks: int, first: int,
                       last: int):
    """(T, N_kv, blocks) int32, the columns that each new token attends to (fhog_paged_block_select)."""
    ext = torch_ext()
    if ext is not None:
        return ext.paged_block_select(q, key_means, page_table, lengths, query_offsets, page_size, blocks, first, last)
    if q.ndim != 3:
        raise ValueError(f"expected a (T, N, H) query, got {tuple(q.shape)}")
    if key_means.ndim != 3 or key_means.shape[2] != q.shape[2]:
        raise ValueError(f"expected (pages, kv_heads, head_dim) key_means for query{tuple(q.shape)}, got {tuple(key_means.shape)}")
    _check_key_means(key_means, ("query", q), key_means.shape)
    page_table, lengths, query_offsets = _check_index(("query", q), page_table, lengths, query_offsets)
    if q.dtype not in DTYPE_CODES:
        raise ValueError(f"unsupported dtype {q.dtype}")
    T, N, Hd = q.shape
    pages, Nk, _ = key_means.shape
    B, width = page_table.shape
    q = q.contiguous()
    if not 1 <= blocks <= 32768:
        raise ValueError(f"blocks must be 1 to 32768, got {blocks}")
    if first < 0 or last < 1 or first + last > blocks:
        raise ValueError(f"needs first >= 0, last >= 1 and first + last <= blocks, got {first}, {last} and {blocks}")
    chosen = torch.empty((T, Nk, blocks), device=q.device, dtype=torch.int32)
    with _on_device(q.device):
        size = lib().fhog_paged_block_select_workspace_bytes(B, T, int(query_offsets is None), Nk, Hd, width, first, last)
        ws = torch.empty(size, device=q.device, dtype=torch.uint8) if size else None
        check(lib().fhog_paged_block_select(
            _stream(q.device), _ptr(q), _ptr(key_means), _ptr(page_table), _ptr(lengths), _ptr(query_offsets), _ptr(chosen),
            _ptr(ws), size, B, T, N, Nk, Hd, pages, page_size, width, DTYPE_CODES[q.dtype], blocks, first, last))
    return chosen


def paged_block_attention(q, chosen, k_cache, v_cache, page_table, lengths, query_offsets, k_scale, v_scale, scale: float,
                          out=None):
    """out (T, N, H) of the packed new tokens q over the chosen (T, N_kv, blocks) columns of a paged cache
    (fhog_paged_block_attention)."""
    ext = torch_ext()
    if ext is not None:
        return ext.paged_block_attention(q, chosen, k_cache, v_cache, page_table, lengths, query_offsets, k_scale, v_scale,
                                         float(scale), out)
    if q.ndim != 3:
        raise ValueError(f"expected a (T, N, H) query, got {tuple(q.shape)}")
    (pages, Nk, page, Hd, B, width), page_table, lengths, query_offsets = _check_cache(
        ("query", q), k_cache, v_cache, page_table, lengths, query_offsets, k_scale, v_scale, q.dtype)
    T, N, Hq = q.shape
    if Hq != Hd:
        raise ValueError(f"query{tuple(q.shape)} and key_cache{tuple(k_cache.shape)} disagree on head_dim")
    if q.dtype not in DTYPE_CODES:
        raise ValueError(f"unsupported dtype {q.dtype}")
    _check_inputs([("query", q), ("blocks", chosen)])
    if chosen.ndim != 3 or tuple(chosen.shape[:2]) != (T, Nk) or chosen.dtype != torch.int32:
        raise ValueError(f"blocks must be torch.int32 {(T, Nk, 'blocks')}, got {tuple(chosen.shape)} of {chosen.dtype}")
    clear = out is None
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    else:
        _check_inputs([("query", q), ("out", out)], q.dtype)
        _expect("out", out, q.shape)
        if not out.is_contiguous():
            raise ValueError("out must be contiguous")
    q, chosen = _contig(q, chosen)
    if not clear:
        _check_apart(out, "query", q)
        _check_apart(out, "blocks", chosen)
        _check_apart_from("out", out, k_cache, v_cache, k_scale, v_scale, page_table, lengths, query_offsets)
    with _on_device(q.device):
        size = lib().fhog_paged_block_workspace_bytes(B, T, int(query_offsets is None), N, Nk, Hd, page, width,
                                                      chosen.shape[2])
        ws = torch.empty(size, device=q.device, dtype=torch.uint8) if size else None
        check(lib().fhog_paged_block_attention(
            _stream(q.device), _ptr(q), _ptr(chosen), _ptr(k_cache), _ptr(v_cache), _ptr(k_scale), _ptr(v_scale),
            _ptr(page_table), _ptr(lengths), _ptr(query_offsets), _ptr(out), _ptr(ws), size, B, T, N, Nk, Hd, pages, page,
            width, DTYPE_CODES[q.dtype], CACHE_DTYPE_CODES[k_cache.dtype], chosen.shape[2], int(clear), float(scale)))
    if not clear:
        _written(out)
    return out


# ------------------------------------------------- norms with rotation

def _rows(t):
    """t with its rows (last axis) contiguous; elements between rows may be any."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


class _RotaryCall:
    """The checked arguments that the three calls share: q (B, T, N, H) and k (B, T, Nk, H) (any strides
    between rows), weights (H,) or None, frequencies (R / 2,) fp32 or None, positions (T,) or (B, T) or
    lengths (sequences,) [and query_offsets (sequences + 1,)] with B = 1 or neither, eps None: no norms.
    like: tensors of q's and k's shapes that stand for them where the rows themselves are not read."""

    def __init__(self, q, k, wq, wk, frequencies, positions, lengths, query_offsets, interleaved, eps, strided=True):
        named = [("query", q), ("key", k)]
        index = [(n, t) for n, t in (("positions", positions), ("lengths", lengths), ("query_offsets", query_offsets))
                 if t is not None]
        weights = [(n, t) for n, t in (("query_weight", wq), ("key_weight", wk)) if t is not None]
        freq = [] if frequencies is None else [("frequencies", frequencies)]
        _check_inputs(named + weights + freq + index)
        _check_inputs(named, q.dtype)
        if q.dtype not in DTYPE_CODES:
            raise ValueError(f"unsupported dtype {q.dtype}")
        if q.ndim != 4 or k.ndim != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
            raise ValueError("expected query (B, T, N, H) and key (B, T, N_kv, H) of the same tokens and head_dim, got "
                             f"{tuple(q.shape)} and {tuple(k.shape)}")
        B, T, N, Hd = q.shape
        if eps is None and weights:
            raise ValueError("weights need norms (eps is None)")
        weight_dtype = weights[0][1].dtype if weights else q.dtype
        for name, t in weights:
            _expect(name, t, (Hd,), weight_dtype)
        if weight_dtype not in (q.dtype, torch.float32):
            raise ValueError(f"weights must be of {q.dtype} or torch.float32, got {weight_dtype}")
        if frequencies is not None:
            if frequencies.ndim != 1 or 2 * frequencies.shape[0] > Hd or frequencies.dtype != torch.float32:
                raise ValueError(f"frequencies must be torch.float32 (R / 2,) with R <= head_dim, got "
                                 f"{tuple(frequencies.shape)} of {frequencies.dtype} for head_dim {Hd}")
        if positions is not None:
            if lengths is not None:
                raise ValueError("positions and lengths exclude each other")
            if positions.dtype not in (torch.int32, torch.int64):
                raise ValueError(f"positions has dtype {positions.dtype}, expected torch.int32 or torch.int64")
            if tuple(positions.shape) not in ((T,), (B, T)):
                raise ValueError(f"positions has shape {tuple(positions.shape)}, expected {(T,)} or {(B, T)}")
        if query_offsets is not None and lengths is None:
            raise ValueError("query_offsets needs lengths")
        if lengths is not None:
            if lengths.ndim != 1:
                raise ValueError(f"expected (batch,) lengths, got {tuple(lengths.shape)}")
            if B != 1:
                raise ValueError(f"lengths go with packed tokens (T, N, H), got a batch of {B}")
            if query_offsets is None:
                _expect("lengths", lengths, (T,))
            else:
                _expect("query_offsets", query_offsets, (lengths.shape[0] + 1,))
            for name, t in index:
                if t.dtype != torch.int32:
                    raise ValueError(f"{name} has dtype {t.dtype}, expected torch.int32")
        self.q, self.k = (_rows(q), _rows(k)) if strided else (q, k)
        contiguous = lambda t: None if t is None else t.contiguous()
        self.wq, self.wk = contiguous(wq), contiguous(wk)
        self.held = tuple(map(contiguous, (frequencies, positions, lengths, query_offsets)))
        frequencies, positions, lengths, query_offsets = self.held
        self.device, self.weight_dtype = q.device, weight_dtype
        self.shape = Rotary(
            B, T, N, k.shape[2], Hd, 0 if frequencies is None else 2 * frequencies.shape[0], DTYPE_CODES[q.dtype],
            DTYPE_CODES[weight_dtype], int(bool(interleaved)), int(eps is not None), 0.0 if eps is None else float(eps),
            0 if positions is None else positions.element_size(),
            0 if positions is None else 1 if positions.ndim == 1 else B, 0 if lengths is None else lengths.shape[0],
            (ctypes.c_longlong * 3)(*self.q.stride()[:3]), (ctypes.c_longlong * 3)(*self.k.stride()[:3]),
            *map(_ptr, self.held))

    def contiguous(self, q_name, q, k_name, k):
        """Tensors of q's and k's shapes, checked."""
        _check_inputs([("query", self.q), (q_name, q), (k_name, k)], self.q.dtype)
        _expect(q_name, q, self.q.shape)
        _expect(k_name, k, self.k.shape)
        return _contig(q, k)

    def rows(self):
        return tuple(torch.empty(t.shape, device=self.device, dtype=t.dtype) for t in (self.q, self.k))

    def weights(self):
        return tuple(None if w is None else torch.empty_like(w) for w in (self.wq, self.wk))

    def workspace(self):
        if self.wq is None and self.wk is None:
            return None
        size = lib().fhog_qk_norm_rotary_workspace_bytes(ctypes.byref(self.shape))
        return torch.empty(size, device=self.device, dtype=torch.uint8) if size else None


def qk_norm_rotary_fwd(q, k, wq, wk, frequencies, positions, lengths, query_offsets, interleaved, eps):
    """(q_out, k_out), contiguous (fhog_qk_norm_rotary_fwd; the arguments: _RotaryCall)."""
    c = _RotaryCall(q, k, wq, wk, frequencies, positions, lengths, query_offsets, interleaved, eps)
    out = c.rows()
    with _on_device(c.device):
        check(lib().fhog_qk_norm_rotary_fwd(_stream(c.device), ctypes.byref(c.shape), _ptr(c.q), _ptr(c.k), _ptr(c.wq),
                                            _ptr(c.wk), *map(_ptr, out)))
    return out


def qk_norm_rotary_bwd(q, k, wq, wk, gq, gk, frequencies, positions, lengths, query_offsets, interleaved, eps):
    """(dq, dk, dwq, dwk) from the cotangents gq, gk of the forward's results; None where a weight is.
    Without norms q and k are only looked at for their shapes."""
    c = _RotaryCall(q, k, wq, wk, frequencies, positions, lengths, query_offsets, interleaved, eps, eps is not None)
    gq, gk = c.contiguous("query's cotangent", gq, "key's cotangent", gk)
    d, dw = c.rows(), c.weights()
    with _on_device(c.device):
        ws = c.workspace()
        x = (None, None) if eps is None else (_ptr(c.q), _ptr(c.k))
        check(lib().fhog_qk_norm_rotary_bwd(_stream(c.device), ctypes.byref(c.shape), *x, _ptr(c.wq), _ptr(c.wk),
                                            _ptr(gq), _ptr(gk), *map(_ptr, d), *map(_ptr, dw), _ptr(ws)))
    return (*d, *dw)


def qk_norm_rotary_bwdbwd(q, k, wq, wk, gq, gk, uq, uk, zq, zk, frequencies, positions, lengths, query_offsets,
                          interleaved, eps):
    """Cotangents (dq2, dk2, dwq2, dwk2, dgq, dgk) of the backward's inputs from those (uq, uk, zq, zk) of its
    results; norms only."""
    c = _RotaryCall(q, k, wq, wk, frequencies, positions, lengths, query_offsets, interleaved, eps)
    gq, gk = c.contiguous("query's cotangent", gq, "key's cotangent", gk)
    uq, uk = c.contiguous("cotangent of query's gradient", uq, "cotangent of key's gradient", uk)
    z = []
    for w, t in ((c.wq, zq), (c.wk, zk)):
        if w is not None:
            _check_inputs([("query", c.q), ("cotangent of a weight's gradient", t)])
            _expect("cotangent of a weight's gradient", t, w.shape, w.dtype)
        z.append(None if w is None else t.contiguous())
    d2, dg, dw2 = c.rows(), c.rows(), c.weights()
    with _on_device(c.device):
        ws = c.workspace()
        check(lib().fhog_qk_norm_rotary_bwdbwd(
            _stream(c.device), ctypes.byref(c.shape), _ptr(c.q), _ptr(c.k), _ptr(c.wq), _ptr(c.wk), _ptr(gq), _ptr(gk),
            _ptr(uq), _ptr(uk), *map(_ptr, z), *map(_ptr, d2), *map(_ptr, dw2), *map(_ptr, dg), _ptr(ws)))
    return (*d2, *dw2, *dg)
