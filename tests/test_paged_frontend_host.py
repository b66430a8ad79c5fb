"""The paged cache's operators under autograd, without a GPU: forward-mode derivatives, and tensors that
are written to or scale what is read while they require a gradient."""

from __future__ import annotations

import pytest
import torch
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
