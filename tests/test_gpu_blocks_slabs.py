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
