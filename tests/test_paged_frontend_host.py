"""The paged cache's operators under torch's transforms, without a GPU: forward-mode derivatives,
vmap, fake tensors, and tensors that are written to while they require a gradient."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad

import flash_hog

BF16, E4M3, E8M0 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu


def cache(kind=BF16, device="cpu"):
    x = dict(key_cache=torch.zeros(4, 2, 16, 64, dtype=kind, device=device),
             value_cache=torch.zeros(4, 2, 16, 64, dtype=kind, device=device),
             page_table=torch.zeros(3, 2, dtype=torch.int32, device=device),
             lengths=torch.ones(3, dtype=torch.int32, device=device))
    if kind == E4M3:
        x.update({n: torch.zeros(4, 2, 16, dtype=torch.uint8, device=device).view(E8M0)
                  for n in ("key_scale", "value_scale")})
    return x


def rows(heads, device="cpu", dtype=BF16):
    return torch.zeros(3, heads, 64, dtype=dtype, device=device)


def dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("grad_mode", [True, False], ids=["grad", "no_grad"])
def test_forward_mode_is_refused(grad_mode):
    """A dual tensor does not require a gradient, and its tangent would be lost."""
    x, q, k = cache(), rows(4), rows(2)
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        duals = {n: dual(x[n]) for n in ("key_cache", "value_cache")}
        calls = [lambda: flash_hog.paged_attention(dual(q), **x),
                 lambda: flash_hog.paged_cache_write(dual(k), k, **x),
                 lambda: flash_hog.paged_cache_write(k, dual(k), **x),
                 lambda: flash_hog.paged_attention(q, **x, out=dual(q))]
        for n in duals:
            calls += [lambda n=n: flash_hog.paged_attention(q, **{**x, n: duals[n]}),
                      lambda n=n: flash_hog.paged_cache_write(k, k, **{**x, n: duals[n]}),
                      lambda n=n: flash_hog.paged_cache_read(**{**x, n: duals[n]})]
        for i, call in enumerate(calls):
            with pytest.raises(RuntimeError, match="has no derivative"):
                call()
                pytest.fail(f"call {i} was accepted")
        # a level that is entered says nothing about tensors without a tangent
        with pytest.raises(ValueError, match="must be on a GPU device"):
            flash_hog.paged_attention(q, **x)
    with pytest.raises(RuntimeError, match="has no derivative"):
        torch.func.jvp(lambda t: flash_hog.paged_attention(t, **x), (q,), (q,))


def test_written_tensors_that_require_a_gradient_are_refused():
    """out and the scales, as the caches themselves."""
    q, k, x = rows(4), rows(2), cache(E4M3)
    with pytest.raises(RuntimeError, match="has no derivative"):
        flash_hog.paged_attention(q, **x, out=rows(4).requires_grad_(True))
    for n in ("key_scale", "value_scale"):
        changed = {**x, n: torch.zeros(4, 2, 16, dtype=torch.uint8).view(E8M0).requires_grad_(True)}
        for call in (lambda: flash_hog.paged_attention(q, **changed), lambda: flash_hog.paged_cache_write(k, k, **changed),
                     lambda: flash_hog.paged_cache_read(**changed)):
            with pytest.raises(RuntimeError, match="has no derivative"):
                call()
        with torch.no_grad(), pytest.raises(ValueError, match="must be on a GPU device"):
            flash_hog.paged_attention(q, **changed)


def test_vmap_is_refused():
    x, q, k = cache(), rows(4), rows(2)
    two = lambda t: torch.stack([t, t])
    for call in (lambda: torch.func.vmap(lambda t: flash_hog.paged_attention(t, **x))(two(q)),
                 lambda: torch.func.vmap(lambda t: flash_hog.paged_attention(q, **{**x, "lengths": t}))(two(x["lengths"])),
                 lambda: torch.func.vmap(lambda t: flash_hog.paged_cache_write(t, t, **x))(two(k)),
                 lambda: torch.func.vmap(lambda t: flash_hog.paged_cache_read(**{**x, "key_cache": t}))(two(x["key_cache"]))):
        with pytest.raises(RuntimeError, match="vmap"):
            call()


@pytest.mark.parametrize("kind", [BF16, E4M3], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("device", ["cuda", "cpu"])
def test_fake_tensors(device, kind):
    """Shapes and types of all three outside of torch.compile, as dot_product_attention gives them."""
    with FakeTensorMode():
        x, q, k = cache(kind, device), rows(4, device), rows(2, device)
        out = flash_hog.paged_attention(q, **x, window=9, sinks=1)
        assert out.shape == q.shape and out.dtype == BF16 and out.device == q.device
        assert flash_hog.paged_cache_write(k, k, **x) is None
        for t in flash_hog.paged_cache_read(**x, dtype=BF16):
            assert t.shape == (3, 32, 2, 64) and t.dtype == BF16
        with pytest.raises(ValueError, match="out is not supported"):
            flash_hog.paged_attention(q, **x, out=torch.empty_like(q))


def test_tensors_made_under_a_transform():
    """A tensor that torch.func.grad wraps without differentiating it reaches the operators."""
    x, k = cache(device="meta"), rows(2, "meta")

    def loss(w):
        q = torch.zeros(3, 4, 64, dtype=BF16, device="meta")
        flash_hog.paged_cache_write(k * 1, k, **x)
        out = flash_hog.paged_attention(q, **x)
        assert out.shape == q.shape
        return (w * out.detach().float()).sum()

    w = torch.zeros(3, 4, 64, device="meta")
    assert torch.func.grad(loss)(w).shape == w.shape
