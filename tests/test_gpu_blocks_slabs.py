"""paged_block_attention of more tokens than a slab of its workspace holds, with sequences that start behind the first
slab and off a multiple of 64 tokens."""

from __future__ import annotations

import pytest
import torch

import blocks_reference as ref
from test_gpu_blocks import BF16, make, many_lists
from test_gpu_paged import check

pytestmark = pytest.mark.gpu


# 132 KiB a token: slabs of 7936 tokens
@pytest.mark.parametrize("lengths,new", [([6000, 5000, 4000], [5001, 4001, 3001]), ([20001, 200], [20001, 3])], ids=str)
def test_sequences_behind_a_slab(lengths, new, cuda_device):
    """Each sequence like the call of its own: the same bits where its slabs hold the same tokens of it (rows of a tile share
    the steps of their maxima), and all within the tolerance of 64 bits."""
    import flash_hog

    print("[case] sequences behind a slab", new, flush=True)
    case = (8, 4, 64, BF16, False, 64, lengths, new, 64)
    cache, counts, q, moved, where = make(case, cuda_device)
    lists = many_lists(case, cache, counts, "chosen")
    kv = moved["key_cache"], moved["value_cache"]
    got = flash_hog.paged_block_attention(q.to(cuda_device), lists.to(cuda_device), *kv, **where)
    torch.cuda.synchronize()
    first = 0
    for b, n in enumerate(new):
        rows = slice(first, first + n)
        first += n
        own = dict(page_table=where["page_table"][b:b + 1], lengths=where["lengths"][b:b + 1],
                   query_offsets=torch.tensor([0, n], dtype=torch.int32, device=cuda_device))
        one = flash_hog.paged_block_attention(q[rows].to(cuda_device), lists[rows].to(cuda_device), *kv, **own)
        if n > 1000 and (rows.start == 0 or rows.start // 7936 == (rows.stop - 1) // 7936):
            assert torch.equal(got[rows], one)
        if n <= 5001:
            alone = [n if i == b else 0 for i in range(len(new))]
            check(got[rows], ref.attention_dense(q[rows], cache, alone, lists[rows], 0.125))


def test_long_lists_of_many_tokens(cuda_device):
    """Lists of more blocks than a split holds, of more tokens than 1 GiB of parts: a token's bits are those of a call
    of fewer tokens (a workgroup has one token's rows), and the padded rows behind the last sequence stay."""
    import flash_hog

    print("[case] long lists of many tokens", flush=True)
    length, new, rows = 33000, 32500, 33000
    cache, _, _, moved, where = make((4, 4, 64, BF16, False, 16, [length], [new]), cuda_device)
    kv = moved["key_cache"], moved["value_cache"]
    q = torch.randn((rows, 4, 64), generator=torch.Generator().manual_seed(8)).to(BF16).to(cuda_device)
    lists = (3 * torch.arange(600, dtype=torch.int32) + torch.arange(rows, dtype=torch.int32)[:, None, None] % 3).repeat(1, 4, 1)
    lists = lists.to(cuda_device)
    out = torch.full_like(q, 7.0)
    flash_hog.paged_block_attention(q, lists, *kv, **where, out=out)
    torch.cuda.synchronize()
    assert (out[new:] == 7).all()
    for first, last in ((0, 400), (31000, 32500)):
        own = {**where, "lengths": where["lengths"] - (new - last), "query_offsets": where["query_offsets"] * 0}
        own["query_offsets"][1] = last - first
        assert torch.equal(flash_hog.paged_block_attention(q[first:last], lists[first:last], *kv, **own), out[first:last])
    for t in (0, 31774, 31775, 32499):  # (31775 tokens a slab)
        cache.lengths = [length - new + t + 1]
        want = ref.attention(q[t:t + 1].cpu(), cache, [1], lists[t:t + 1].cpu(), 0.125)
        check(out[t:t + 1], want)
