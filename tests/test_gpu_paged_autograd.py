"""What the paged cache's operators write, as torch's autograd sees it: a tensor that a graph saved
before it was written to must not be used by that graph's backward."""

from __future__ import annotations

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(params=[False, True], ids=["extension", "python"])
def flash_hog(request, monkeypatch):
    import flash_hog
    from flash_hog import _hip

    if request.param:
        monkeypatch.setattr(_hip, "torch_ext", lambda: None)
    return flash_hog


def inputs(device, quantised=False):
    x = ref.Cache([20, 3], 16, 2, 64, BF16, quantised).on(device)
    q, k = (torch.ones((2, n, 64), dtype=BF16, device=device) for n in (4, 2))
    return x, q, k


@pytest.mark.parametrize("quantised", [False, True], ids=["plain", "e4m3"])
def test_written_tensors_have_a_new_version(quantised, flash_hog, cuda_device):
    x, q, k = inputs(cuda_device, quantised)
    out = torch.empty_like(q)
    tensors = {**x, "query": q, "key": k, "out": out}
    caches = [n for n in x if n.endswith(("cache", "scale"))]

    def changed(call):
        before = {n: t._version for n, t in tensors.items()}
        call()
        return [n for n, t in tensors.items() if t._version != before[n]]

    assert changed(lambda: flash_hog.paged_cache_write(k, k, **x)) == caches
    assert changed(lambda: flash_hog.paged_attention(q, **x)) == []
    assert changed(lambda: flash_hog.paged_attention(q, **x, out=out)) == ["out"]
    assert changed(lambda: flash_hog.paged_cache_read(**x)) == []


def test_backward_on_overwritten_tensors_raises(flash_hog, cuda_device):
    x, q, k = inputs(cuda_device)
    out = torch.zeros_like(q)
    for saved, write in ((x["key_cache"], lambda: flash_hog.paged_cache_write(k, k, **x)),
                         (x["value_cache"][0], lambda: flash_hog.paged_cache_write(k, k, **x)),  # a view of it
                         (out, lambda: flash_hog.paged_attention(q, **x, out=out))):
        w = torch.ones((), dtype=BF16, device=cuda_device, requires_grad=True)
        y = (w * saved).sum()
        write()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


def test_inference_tensors_are_written_in_any_mode(flash_hog, cuda_device):
    """A cache made under inference_mode has no version; graphs cannot save it."""
    with torch.inference_mode():
        x, q, k = inputs(cuda_device)
        out = torch.zeros_like(q)
        flash_hog.paged_cache_write(k, k, **x)
        flash_hog.paged_attention(q, **x, out=out)
        want = out.clone()
        out.zero_()
    with torch.no_grad():
        flash_hog.paged_cache_write(k.clone(), k.clone(), **x)
        flash_hog.paged_attention(q.clone(), **x, out=out)
    assert torch.equal(out, want) and bool((want[0] != 0).any())
    plain, _, _ = inputs(cuda_device)
    with torch.inference_mode():  # and one made outside of it keeps its version
        before = plain["key_cache"]._version
        flash_hog.paged_cache_write(k, k, **plain)
    assert plain["key_cache"]._version > before
