"""An out of paged_attention that shares memory with what the kernels read: query itself is replaced
in place, anything else is refused. Rows of one workgroup would otherwise change what another reads."""

from __future__ import annotations

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16

# (heads, kv_heads, head_dim, lengths, new): tokens with and without splits, narrow and wide chunks
SIZES = [(4, 2, 64, [20, 3], None), (4, 1, 128, [5000, 77], None), (12, 3, 64, [300, 40], [200, 40]),
         (32, 8, 128, [2100, 2000], [2100, 1900])]


@pytest.fixture(params=[False, True], ids=["extension", "python"])
def flash_hog(request, monkeypatch):
    import flash_hog
    from flash_hog import _hip

    if request.param:
        monkeypatch.setattr(_hip, "torch_ext", lambda: None)
    return flash_hog


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_out_is_query_or_apart(size, flash_hog, cuda_device):
    heads, kv_heads, d, lengths, new = size
    print("[case] overlap", size, flush=True)
    x = ref.Cache(lengths, 16, kv_heads, d, BF16, False).on(cuda_device)
    total = len(lengths) if new is None else sum(new)
    if new is not None:
        x["query_offsets"] = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=cuda_device)
    buffer = torch.randn(total + 1, heads, d, generator=torch.Generator().manual_seed(3)).to(BF16).to(cuda_device)
    q = buffer[:-1]
    want = flash_hog.paged_attention(q, **x)
    with pytest.raises(ValueError, match="out overlaps query"):
        flash_hog.paged_attention(q, **x, out=buffer[1:])
    with pytest.raises(ValueError, match="out overlaps query"):
        flash_hog.paged_attention(buffer[1:], **x, out=q)
    for n in ("key_cache", "value_cache"):
        room = x[n].new_zeros(total * heads * d + x[n].numel() // 2)  # out's end in a cache's half
        room = torch.cat([room, x[n].flatten()])
        shared = {**x, n: room[-x[n].numel():].view(x[n].shape)}
        at = room.numel() - x[n].numel() - total * heads * d
        free = room[at:at + total * heads * d].view(q.shape)
        assert torch.equal(flash_hog.paged_attention(q, **shared, out=free), want)  # a neighbour's memory
        with pytest.raises(ValueError, match=f"out overlaps {n}"):
            flash_hog.paged_attention(q, **shared, out=room[at + 64:at + 64 + total * heads * d].view(q.shape))
    strided = buffer.new_empty(total, 2 * heads, d)  # read from a copy: no overlap by then
    strided[:, ::2] = q
    flat = strided.view(-1)[:total * heads * d].view(q.shape)
    assert torch.equal(flash_hog.paged_attention(strided[:, ::2], **x, out=flat), want)
    assert torch.equal(flash_hog.paged_attention(q, **x, out=q), want) and torch.equal(q, want)
