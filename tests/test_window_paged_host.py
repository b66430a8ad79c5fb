"""Windowed attention and the paged cache, without a GPU: what the C ABI and the front-end refuse
(before anything reaches a device), workspace sizes, shapes on meta tensors, and the launch
rules that split work."""

from __future__ import annotations

import pytest
import torch

import flash_hog
from flash_hog import _hip
from flash_hog.torch.attention import _effective_window

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def lib():
    return _hip.lib()


def meta(*shape, dtype=BF16):
    return torch.empty(*shape, device="meta", dtype=dtype)


# ------------------------------------------------------------------ the C ABI: windows

def _window_args(pointers, workspace=16, ptr=16, batch=1, n_q=200, n_k=200, heads=1, kv_heads=1, head_dim=64, dtype=2,
                 causal=1, window=8, sinks=2, scale=0.125):
    ws = [] if workspace == "none" else [workspace]
    return [None] + [ptr] * pointers + ws + [batch, n_q, n_k, heads, kv_heads, head_dim, dtype, causal, window, sinks,
                                             scale]


WINDOW_CALLS = {"fhog_window_attention_fwd": (5, "none"), "fhog_window_attention_bwd": (10, 16),
                "fhog_window_attention_bwdbwd": (16, 16)}
WINDOW_REFUSALS = [
    (dict(ptr=None), 1, "q is null"),
    (dict(ptr=8), 1, "not 16-byte aligned"),
    (dict(causal=0), 1, "a window needs causal"),
    (dict(causal=3), 1, "causal must be"),
    (dict(window=0), 1, "window must be >= 1"),
    (dict(window=-(1 << 31)), 1, "window must be >= 1"),
    (dict(sinks=-1), 1, "sinks must be >= 0"),
    (dict(batch=0), 1, "sizes must be >= 1"),
    (dict(n_k=0), 1, "sizes must be >= 1"),
    (dict(heads=3, kv_heads=2), 1, "multiple of kv_heads"),
    (dict(dtype=3), 1, "unknown dtype"),
    (dict(head_dim=96), 2, "head_dim must be 64, 128 or 256"),
    (dict(head_dim=256, dtype=0), 2, "fp32 head_dim must be 64 or 128"),
    (dict(scale=float("nan")), 1, "scale must be finite"),
    (dict(scale=0.0), 2, "scale must be nonzero"),
    (dict(n_q=(1 << 31) - 1, n_k=1), 1, "problem too large"),
    (dict(batch=1 << 20, heads=1 << 10, kv_heads=1), 1, "problem too large"),
]


@pytest.mark.parametrize("name", WINDOW_CALLS)
@pytest.mark.parametrize("kwargs,status,needle", WINDOW_REFUSALS)
def test_window_refusals(lib, name, kwargs, status, needle):
    pointers, workspace = WINDOW_CALLS[name]
    assert getattr(lib, name)(*_window_args(pointers, workspace, **kwargs)) == status
    message = lib.fhog_last_error().decode()
    assert needle in message and message.startswith(name)


@pytest.mark.parametrize("name", ["fhog_window_attention_bwd", "fhog_window_attention_bwdbwd"])
@pytest.mark.parametrize("workspace", [None, 8])
def test_window_needs_its_workspace(lib, name, workspace):
    pointers, _ = WINDOW_CALLS[name]
    args = dict(n_q=1000, n_k=1000, window=8, sinks=2)
    assert lib.fhog_window_workspace_bytes(1, 1000, 1000, 1, 1, 64, 2, 1, 8, 2) > 0
    assert getattr(lib, name)(*_window_args(pointers, workspace, **args)) == 1
    assert "workspace is null or not 16-byte aligned" in lib.fhog_last_error().decode()


def test_window_workspace_bytes(lib):
    def size(batch=1, n_q=1000, n_k=1000, heads=4, kv_heads=2, head_dim=64, dtype=2, causal=1, window=8, sinks=2):
        return lib.fhog_window_workspace_bytes(batch, n_q, n_k, heads, kv_heads, head_dim, dtype, causal, window, sinks)

    part = 2 * 2 * 2 * 64 * 4  # pairs, sinks, dV and dK, columns, fp32
    assert size() >= 2 * part and size() % part == 0  # the sinks' own blocks and at least one chunk
    assert size(sinks=0) == 0
    assert size(window=1000) == 0                    # every query sees its sinks through the window
    assert size(window=(1 << 31) - 1, sinks=(1 << 31) - 1) == 0
    assert size(batch=3) % (3 * part) == 0
    for bad in (dict(window=0), dict(sinks=-1), dict(causal=0), dict(n_q=0), dict(head_dim=65)):
        assert size(**bad) == 0
    # never more than twice the keys' own gradients would take in fp32
    for n in (100, 1000, 5000, 70000, 1 << 20):
        for window in (1, 30, 500, 4096):
            for sinks in (1, 4, 70, 1000, n):
                most = 2 * 2 * n * 2 * 64 * 4 + 2 * part * max(1, sinks)
                assert size(n_q=n, n_k=n, window=window, sinks=sinks) <= most, (n, window, sinks)


# ------------------------------------------------------------------ the C ABI: paged cache

def _paged_args(kind, ptr=16, scale_ptr=16, table=16, offsets=16, workspace=16, workspace_bytes=1 << 40, batch=2,
                total=40, heads=4, kv_heads=2, head_dim=64, num_pages=9, page_size=16, pages_per_seq=4, dtype=2,
                cache_dtype=2, window=0, sinks=0, scale=0.125, max_length=64):
    caches = [ptr, ptr, scale_ptr, scale_ptr]
    if kind == "attention":
        return [None, ptr, *caches, table, table, offsets, ptr, workspace, workspace_bytes, batch, total, heads,
                kv_heads, head_dim, num_pages, page_size, pages_per_seq, dtype, cache_dtype, window, sinks, 1, scale]
    if kind == "write":
        return [None, ptr, ptr, *caches, table, table, offsets, batch, total, kv_heads, head_dim, num_pages, page_size,
                pages_per_seq, dtype, cache_dtype]
    return [None, *caches, table, table, ptr, ptr, batch, max_length, kv_heads, head_dim, num_pages, page_size,
            pages_per_seq, dtype, cache_dtype]


PAGED_CALLS = {"attention": "fhog_paged_attention", "write": "fhog_paged_cache_write", "read": "fhog_paged_cache_read"}
ALL, ROWS, ATTENTION = ("attention", "write", "read"), ("attention", "write"), ("attention",)
PAGED_REFUSALS = [
    (ALL, dict(ptr=None), 1, "is null or not 16-byte aligned"),
    (ALL, dict(ptr=8), 1, "not 16-byte aligned"),
    (ALL, dict(table=None), 1, "page_table is null"),
    (ALL, dict(table=2), 1, "not 4-byte aligned"),
    (ROWS, dict(offsets=2), 1, "query_offsets is not 4-byte aligned"),
    (ROWS, dict(offsets=None), 1, "without query_offsets there is one row a sequence: 40 rows, 2 sequences"),
    (ALL, dict(cache_dtype=3, scale_ptr=None), 1, "an e4m3 cache needs k_scale and v_scale"),
    (ALL, dict(batch=-1), 1, "must not be negative"),
    (ROWS, dict(total=-1), 1, "must not be negative"),
    (("read",), dict(max_length=-1), 1, "must not be negative"),
    (ALL, dict(num_pages=0), 1, "sizes must be >= 1"),
    (ALL, dict(pages_per_seq=0), 1, "sizes must be >= 1"),
    (ALL, dict(kv_heads=0), 1, "sizes must be >= 1"),
    (ATTENTION, dict(heads=3), 1, "multiple of kv_heads"),
    (ALL, dict(page_size=8), 1, "page_size must be a power of two >= 16"),
    (ALL, dict(page_size=24), 1, "page_size must be a power of two >= 16"),
    (ALL, dict(dtype=0, cache_dtype=0), 2, "dtype must be bf16 or fp16"),
    (ALL, dict(dtype=3, cache_dtype=3), 2, "dtype must be bf16 or fp16"),
    (ALL, dict(cache_dtype=1), 2, "the cache must be of dtype 2 or e4m3"),
    (ALL, dict(head_dim=96), 2, "head_dim must be 64, 128 or 256"),
    (ALL, dict(pages_per_seq=1 << 27), 1, "problem too large"),
    (ALL, dict(batch=1 << 24), 1, "problem too large"),
    (ROWS, dict(total=(1 << 31) - 1), 1, "problem too large"),
    (("read",), dict(max_length=(1 << 31) - 1), 1, "problem too large"),
    (ATTENTION, dict(window=-1), 1, "window must be >= 1 (or 0: none)"),
    (ATTENTION, dict(sinks=1), 1, "0 without a window"),
    (ATTENTION, dict(window=4, sinks=-1), 1, "sinks >= 0"),
    (ATTENTION, dict(scale=float("inf")), 1, "scale must be finite"),
    (ATTENTION, dict(scale=0.0), 2, "scale must be nonzero"),
    (ATTENTION, dict(batch=0), 1, "rows without a sequence"),
    (ATTENTION, dict(batch=1, total=1, pages_per_seq=4096, workspace=None), 1, "workspace is null"),
    (ATTENTION, dict(batch=1, total=1, pages_per_seq=4096, workspace_bytes=16), 1, "below its"),
    (ATTENTION, dict(batch=(1 << 24) - 1, kv_heads=4), 1, "problem too large"),
]


@pytest.mark.parametrize("kind,kwargs,status,needle",
                         [(kind, kw, status, needle) for kinds, kw, status, needle in PAGED_REFUSALS for kind in kinds])
def test_paged_refusals(lib, kind, kwargs, status, needle):
    assert getattr(lib, PAGED_CALLS[kind])(*_paged_args(kind, **kwargs)) == status
    message = lib.fhog_last_error().decode()
    assert needle in message and message.startswith(PAGED_CALLS[kind])


def test_paged_calls_without_work(lib):
    """No rows or no sequences: done before a pointer is looked at."""
    for kind, kw in (("attention", dict(total=0)), ("write", dict(total=0)), ("write", dict(batch=0)),
                     ("read", dict(max_length=0)), ("read", dict(batch=0))):
        assert getattr(lib, PAGED_CALLS[kind])(*_paged_args(kind, ptr=None, **kw)) == 0, (kind, kw)


def test_paged_workspace_bytes(lib):
    def size(batch=1, total=1, single=1, heads=8, kv_heads=2, head_dim=128, page_size=16, pages_per_seq=2048, window=0,
             sinks=0):
        return lib.fhog_paged_workspace_bytes(batch, total, single, heads, kv_heads, head_dim, page_size, pages_per_seq,
                                              window, sinks)

    assert size() > 0 and size() % ((128 + 2) * 4) == 0
    assert size(pages_per_seq=1) == 0                       # too short to split
    assert size(window=20) == 0
    assert size(batch=4096, total=4096) == 0                # rows enough without splits
    assert size(batch=2, total=60000, single=0, heads=8) == 0
    for bad in (dict(heads=3), dict(page_size=17), dict(head_dim=32), dict(total=0), dict(window=-1)):
        assert size(**bad) == 0
    # a bounded number of parts, whatever the sizes
    for batch in (1, 3, 16, 100, 1000):
        for pages in (1, 7, 100, 4096, 1 << 22):
            for new in (1, 5, 100, 4000):
                got = size(batch=batch, total=batch * new, single=int(new == 1), pages_per_seq=pages)
                assert got <= 4096 * 128 * (128 + 2) * 4, (batch, pages, new)


# ------------------------------------------------------------------ the front-end

def test_window_arguments_are_checked():
    q = meta(1, 8, 2, 64)
    with pytest.raises(ValueError, match="window needs is_causal"):
        flash_hog.dot_product_attention(q, q, q, window=3)
    for window, sinks in ((0, 0), (-1, 0), (4, -1)):
        with pytest.raises(ValueError, match="window must be >= 1 and sinks >= 0"):
            flash_hog.dot_product_attention(q, q, q, is_causal=True, window=window, sinks=sinks)
    with pytest.raises(ValueError, match="sinks needs a window"):
        flash_hog.dot_product_attention(q, q, q, is_causal=True, sinks=1)
    for window, sinks in ((4.0, 0), (4, 1.5), ("4", 0)):
        with pytest.raises(TypeError):
            flash_hog.dot_product_attention(q, q, q, is_causal=True, window=window, sinks=sinks)
    for args in ((-1, 0), (0, 1), (3, -1)):
        with pytest.raises(ValueError, match="window"):
            _hip._window_args(*args)


def test_effective_window_against_the_mask():
    """(0, 0) exactly where the window hides nothing that the causal mask shows."""
    from window_reference import visible

    for n_q in (1, 5, 12):
        for n_k in (1, 4, 12):
            for alignment in ("top_left", "bottom_right"):
                for window in (1, 3, 8, 11, 12, 13, 50):
                    for sinks in (0, 1, 3, 12, 40):
                        same = torch.equal(visible(n_q, n_k, alignment, window, sinks),
                                           visible(n_q, n_k, alignment, 0, 0))
                        got = _effective_window(n_q, n_k, alignment, window, sinks)
                        assert got in ((0, 0), (window, sinks))
                        assert got == (window, sinks) or same


def test_window_shapes_on_meta_tensors():
    """Shapes through both derivatives, unbatched and padded head dims, vmap and torch.compile."""
    kw = dict(is_causal=True, window=5, sinks=2)
    for d in (64, 40):
        q = meta(2, 30, 4, d).requires_grad_(True)
        k, v = (meta(2, 30, 2, d).requires_grad_(True) for _ in range(2))
        out = flash_hog.dot_product_attention(q, k, v, **kw)
        g = torch.autograd.grad(out, (q, k, v), torch.empty_like(out), create_graph=True)
        h = torch.autograd.grad(g, (q, k, v), tuple(torch.empty_like(t) for t in g))
        assert [t.shape for t in h] == [q.shape, k.shape, v.shape]
    assert flash_hog.dot_product_attention(meta(9, 4, 64), meta(9, 2, 64), meta(9, 2, 64), **kw).shape == (9, 4, 64)

    def attn(q, k, v):
        return flash_hog.dot_product_attention(q, k, v, **kw)

    q, k = meta(3, 2, 30, 4, 64), meta(3, 2, 30, 2, 64)
    assert torch.func.vmap(attn)(q, k, k).shape == q.shape
    assert torch.func.vmap(attn, in_dims=(0, None, None))(q, k[0], k[0]).shape == q.shape
    grads = torch.func.vmap(torch.func.grad(lambda *x: attn(*x).float().sum(), argnums=(0, 1, 2)))(q, k, k)
    assert [t.shape for t in grads] == [q.shape, k.shape, k.shape]
    assert torch.compile(attn, backend="aot_eager", fullgraph=True)(q[0], k[0], k[0]).shape == q[0].shape


def _cache(kind=BF16, **changed):
    x = dict(key_cache=torch.zeros(4, 2, 16, 64, dtype=kind), value_cache=torch.zeros(4, 2, 16, 64, dtype=kind),
             page_table=torch.zeros(3, 2, dtype=torch.int32), lengths=torch.ones(3, dtype=torch.int32))
    x.update(changed)
    return x


@pytest.mark.parametrize("python", [False, True], ids=["extension", "python"])
def test_paged_functions_refuse_host_tensors(python, monkeypatch):
    if python:
        monkeypatch.setattr(_hip, "torch_ext", lambda: None)
    q, k = torch.zeros(3, 4, 64, dtype=BF16), torch.zeros(3, 2, 64, dtype=BF16)
    with pytest.raises(ValueError, match="query must be on a GPU device, got cpu"):
        flash_hog.paged_attention(q, **_cache())
    with pytest.raises(ValueError, match="key must be on a GPU device, got cpu"):
        flash_hog.paged_cache_write(k, k, **_cache())
    with pytest.raises(ValueError, match="key_cache must be on a GPU device, got cpu"):
        flash_hog.paged_cache_read(**_cache())


def test_paged_functions_have_no_derivative():
    q, k = torch.zeros(3, 4, 64, dtype=BF16), torch.zeros(3, 2, 64, dtype=BF16)
    for call in (lambda: flash_hog.paged_attention(q.requires_grad_(True), **_cache()),
                 lambda: flash_hog.paged_cache_write(k.requires_grad_(True), k, **_cache()),
                 lambda: flash_hog.paged_cache_read(**_cache(key_cache=torch.zeros(4, 2, 16, 64).requires_grad_(True)))):
        with pytest.raises(RuntimeError, match="has no derivative"):
            call()


def test_paged_window_arguments_are_checked():
    q = torch.zeros(3, 4, 64, dtype=BF16)
    for window, sinks in ((0, 0), (-3, 0), (4, -1)):
        with pytest.raises(ValueError, match="window must be >= 1 and sinks >= 0"):
            flash_hog.paged_attention(q, **_cache(), window=window, sinks=sinks)
    with pytest.raises(ValueError, match="sinks needs a window"):
        flash_hog.paged_attention(q, **_cache(), sinks=2)
    with pytest.raises(TypeError):
        flash_hog.paged_attention(q, **_cache(), window=2.5)
    with pytest.raises(ValueError, match="page_table"):
        flash_hog.paged_cache_read(**_cache(page_table=torch.zeros(3, dtype=torch.int32)))


def test_paged_operators_trace():
    """torch.compile takes all three as operators (fake kernels on meta tensors)."""
    x = {n: t.to("meta") for n, t in _cache().items()}

    def step(q, k, v):
        flash_hog.paged_cache_write(k, v, **x)
        out = flash_hog.paged_attention(q, **x, window=9, sinks=1)
        return out, flash_hog.paged_cache_read(**x)

    q, k = meta(3, 4, 64), meta(3, 2, 64)
    out, (kd, vd) = torch.compile(step, backend="aot_eager", fullgraph=True)(q, k, k)
    assert out.shape == q.shape and kd.shape == vd.shape == (3, 32, 2, 64) and kd.dtype == BF16
