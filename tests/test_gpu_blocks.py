"""paged_key_means, paged_block_select and paged_block_attention against plain 64-bit forms.

Means are one rounding of a sum that is exact in 64 bits, and choices are whole numbers: both are compared
for equality. Attention: test_gpu_paged.py's tolerance (check), fixed there for the same roundings.
"""

from __future__ import annotations

import pytest
import torch

import blocks_reference as ref
import paged_reference
from test_gpu_paged import check

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16

# (heads, kv_heads, head_dim, dtype, quantised, page, lengths, new (None: one each), blocks, first, last)
CASES = [
    (1, 1, 64, BF16, False, 16, [1], None, 1, 0, 1),
    (4, 2, 64, BF16, False, 16, [1, 15, 16, 17, 0, 33, 200, 700], None, 4, 1, 1),
    (4, 2, 64, BF16, False, 16, [1000], None, 7, 2, 2),           # an odd number of half tiles
    (12, 4, 64, FP16, False, 32, [70, 331, 1111], None, 5, 0, 1),
    (8, 1, 128, BF16, False, 64, [5, 500, 3000], None, 6, 1, 2),
    (34, 2, 64, BF16, False, 16, [400, 777], None, 9, 1, 1),      # 17 heads a group
    (4, 4, 256, BF16, False, 16, [100, 2570], None, 8, 1, 1),
    (8, 2, 128, BF16, True, 64, [1, 64, 65, 4000], None, 16, 1, 1),
    (8, 2, 64, FP16, True, 16, [3, 90, 700], None, 11, 3, 1),
    (4, 2, 256, FP16, True, 128, [129, 2000], None, 4, 1, 3),
    (4, 1, 128, BF16, False, 256, [255, 256, 3000], None, 3, 1, 1),
    (4, 2, 64, BF16, False, 16, [150, 3, 20], [7, 3, 1], 4, 1, 1),
    (2, 2, 64, BF16, False, 16, [150, 3, 0, 200], [150, 2, 0, 33], 3, 1, 1),
    (8, 2, 128, BF16, False, 16, [300, 80], [64, 80], 5, 1, 2),
    (4, 1, 128, FP16, False, 64, [700], [129], 4, 1, 1),
    (2, 1, 256, BF16, False, 16, [150, 90], [70, 20], 6, 0, 2),
    (8, 2, 128, BF16, True, 64, [600, 80], [64, 80], 4, 1, 1),
    (4, 2, 64, FP16, True, 16, [333, 40], [100, 40], 7, 1, 1),
    (6, 2, 64, BF16, False, 16, [3, 2], [5, 2], 4, 1, 1),         # more new tokens than the length: two see nothing
    (3, 3, 64, FP16, True, 64, [520, 1030], [260, 300], 4, 1, 1),
    (32, 4, 64, BF16, False, 32, [400], [200], 6, 1, 1),
    (16, 1, 256, FP16, True, 32, [200], [100], 3, 0, 1),
]


def case_id(c):
    H, Hk, D, dt, q8, page, lengths, new, blocks, first, last = c
    n = "x".join(map(str, lengths))
    return f"h{H}_{Hk}_d{D}_{str(dt)[6:]}{'_e4m3' if q8 else ''}_p{page}_len{n}" + \
        (f"_new{'x'.join(map(str, new))}" if new else "") + f"_b{blocks}_{first}_{last}"


def make(c, device, seed=5, width=None):
    H, Hk, D, dtype, quantised, page, lengths, new = c[:8]
    cache = paged_reference.Cache(lengths, page, Hk, D, dtype, quantised, seed=seed, width=width)
    counts = new or [1] * len(lengths)
    gen = torch.Generator().manual_seed(seed + 1)
    q = torch.randn((sum(counts), H, D), generator=gen).to(dtype)
    moved = cache.on(device)
    where = {"page_table": moved["page_table"], "lengths": moved["lengths"], "query_offsets": None}
    if new:
        offsets = torch.zeros(len(new) + 1, dtype=torch.int32)
        offsets[1:] = torch.cumsum(torch.tensor(new), 0)
        where["query_offsets"] = offsets.to(device)
    return cache, counts, q, moved, where


def scales(moved):
    return {k: v for k, v in moved.items() if "scale" in k}


def all_means(cache):
    """Means of all full pages; NaN elsewhere."""
    shape = cache.cache["k"].shape
    return ref.key_means(cache, cache.lengths, torch.full((shape[0], shape[1], shape[3]), float("nan")))


@pytest.mark.parametrize("case", CASES, ids=case_id)
def test_key_means(case, cuda_device):
    import flash_hog

    print("[case] means", case_id(case), flush=True)
    cache, counts, _, moved, where = make(case, cuda_device)
    shape = cache.cache["k"].shape
    before = torch.randn((shape[0], shape[1], shape[3]), generator=torch.Generator().manual_seed(1))
    means = before.to(cuda_device)
    assert flash_hog.paged_key_means(moved["key_cache"], means, **where, key_scale=moved.get("key_scale")) is None
    assert torch.equal(means.cpu(), ref.key_means(cache, counts, before))


@pytest.mark.parametrize("case", CASES, ids=case_id)
def test_select(case, cuda_device):
    import flash_hog

    print("[case] select", case_id(case), flush=True)
    cache, counts, q, moved, where = make(case, cuda_device)
    blocks, first, last = case[8:]
    means = all_means(cache)
    got = flash_hog.paged_block_select(q.to(cuda_device), means.to(cuda_device), **where, page_size=cache.page, blocks=blocks,
                                       first=first, last=last)
    want = ref.select(q, means, cache.table, cache.lengths, counts, cache.page, blocks, first, last)
    assert got.dtype == torch.int32 and torch.equal(got.cpu(), want)


@pytest.mark.parametrize("case", CASES, ids=case_id)
def test_attention(case, cuda_device):
    import flash_hog

    print("[case] attention", case_id(case), flush=True)
    cache, counts, q, moved, where = make(case, cuda_device)
    blocks, first, last = case[8:]
    chosen = ref.select(q, all_means(cache), cache.table, cache.lengths, counts, cache.page, blocks, first, last)
    for scale in (None, -0.21):
        got = flash_hog.paged_block_attention(q.to(cuda_device), chosen.to(cuda_device), moved["key_cache"],
                                              moved["value_cache"], **where, **scales(moved), scale=scale)
        check(got, ref.attention(q, cache, counts, chosen, scale or q.shape[-1] ** -0.5), case_id(case))


@pytest.mark.parametrize("case", [CASES[1], CASES[3], CASES[8], CASES[13], CASES[19]], ids=case_id)
def test_any_lists(case, cuda_device):
    """Lists in any order, with nothing, columns behind the token or outside the table, and a column twice, which
    counts twice; lists that show nothing give zeros."""
    import flash_hog

    print("[case] any lists", case_id(case), flush=True)
    cache, counts, q, moved, where = make(case, cuda_device)
    gen = torch.Generator().manual_seed(8)
    T, N, width = q.shape[0], case[1], cache.table.shape[1]
    chosen = torch.randint(-1, width + 2, (T, N, 9), generator=gen).to(torch.int32)
    chosen[::3, 0] = -1
    chosen[1::4, :, 3] = 2 ** 31 - 1
    chosen[2::4, :, 4] = -2 ** 31
    got = flash_hog.paged_block_attention(q.to(cuda_device), chosen.to(cuda_device), moved["key_cache"], moved["value_cache"],
                                          **where, **scales(moved))
    check(got, ref.attention(q, cache, counts, chosen, q.shape[-1] ** -0.5), case_id(case))
    assert not got[::3, :case[0] // N].any()


@pytest.mark.parametrize("blocks,page,length", [(600, 16, 20000), (1300, 16, 25000), (520, 32, 20000), (64, 128, 9000)])
def test_many_blocks(blocks, page, length, cuda_device):
    """More blocks than a split lists, and as many as there are."""
    import flash_hog

    case = (4, 1, 64, BF16, False, page, [length, 40], None, blocks, 1, 1)
    print("[case] many blocks", case_id(case), flush=True)
    cache, counts, q, moved, where = make(case, cuda_device)
    means = all_means(cache)
    got = flash_hog.paged_block_select(q.to(cuda_device), means.to(cuda_device), **where, page_size=page, blocks=blocks)
    want = ref.select(q, means, cache.table, cache.lengths, counts, page, blocks, 1, 1)
    assert torch.equal(got.cpu(), want)
    out = flash_hog.paged_block_attention(q.to(cuda_device), got, moved["key_cache"], moved["value_cache"], **where)
    check(out, ref.attention(q, cache, counts, want, 0.125))
    # all of the pages are all of the keys
    if blocks * page >= length:
        check(out, flash_hog.paged_attention(q.to(cuda_device), moved["key_cache"], moved["value_cache"], **where).cpu())


def choose(means, q, page, blocks, length, device, first=0, last=1, table=None, tiles=False):
    """The lists of one token; tiles: as the last of so many that sixteen share a workgroup."""
    import flash_hog

    pages = means.shape[0]
    table = torch.arange(pages, dtype=torch.int32)[None] if table is None else table
    if tiles:
        offsets = torch.tensor([0, 4096], dtype=torch.int32, device=device)
        return flash_hog.paged_block_select(q.to(device).expand(4096, -1, -1), means.to(device), table.to(device),
                                            torch.tensor([length], dtype=torch.int32, device=device), offsets,
                                            page_size=page, blocks=blocks, first=first, last=last)[-1].cpu()
    return flash_hog.paged_block_select(q.to(device), means.to(device), table.to(device),
                                        torch.tensor([length], dtype=torch.int32, device=device), page_size=page,
                                        blocks=blocks, first=first, last=last).cpu()[0]


@pytest.mark.parametrize("head_dim,dtype", [(64, BF16), (128, FP16), (256, BF16)])
@pytest.mark.parametrize("width", [None, 300, 514, 1027, 1028])
def test_select_many(width, head_dim, dtype, cuda_device):
    """So many tokens that sixteen share a workgroup; sequences of one token, so many that scores go through memory."""
    import flash_hog

    print("[case] select many", head_dim, width, flush=True)
    gen = torch.Generator().manual_seed(6)
    for lengths, new in (([3000, 700, 16, 2049], [1000, 400, 16, 700]), (torch.randint(0, 3000, (300,), generator=gen).tolist(), None)):
        counts = new or [1] * len(lengths)
        pages, batch, T, cols = 500, len(lengths), sum(counts), width or -(-max(lengths) // 16)
        means = torch.randn((pages, 4, head_dim), generator=gen)
        q = torch.randn((T, 8, head_dim), generator=gen).to(dtype)
        # (random pages: one twice in a row ties)
        table = torch.randint(-2, pages + 2, (batch, cols), generator=gen).to(torch.int32)
        offsets = torch.zeros(batch + 1, dtype=torch.int32)
        offsets[1:] = torch.tensor(counts).cumsum(0)
        for blocks, first, last in ((20, 2, 1), (3, 1, 2), (260, 0, 3)):
            got = flash_hog.paged_block_select(
                q.to(cuda_device), means.to(cuda_device), table.to(cuda_device), torch.tensor(lengths, dtype=torch.int32, device=cuda_device),
                None if new is None else offsets.to(cuda_device), page_size=16, blocks=blocks, first=first, last=last)
            assert torch.equal(got.cpu(), ref.select_dense(q, means, table, lengths, counts, 16, blocks, first, last)), (blocks, new is None)


@pytest.mark.parametrize("case", [CASES[i] for i in (0, 1, 3, 8, 12, 18)], ids=case_id)
def test_select_oracles_agree(case, cuda_device):
    cache, counts, q, *_ = make(case, "cpu")
    blocks, first, last = case[8:]
    args = (q, all_means(cache), cache.table, cache.lengths, counts, cache.page, blocks, first, last)
    assert torch.equal(ref.select(*args), ref.select_dense(*args))


@pytest.mark.parametrize("width", [None, 300, 514, 1027, 1028, 3000])
@pytest.mark.parametrize("new", [[1, 40, 16, 5], [130, 1, 0, 33], [2, 9, 1, 3]], ids=str)
def test_select_tiles_and_tokens(new, width, cuda_device):
    """Sequences with many and with few new tokens, and tables as wide as the rules tell apart: scores in LDS, and in
    memory with tiles of 16 tokens that end anywhere."""
    import flash_hog

    lengths = [3000, 700, 16, 2049]
    case = (4, 2, 64, BF16, False, 16, lengths, new, 20, 2, 1)
    print("[case] tiles", case_id(case), width, flush=True)
    cache, counts, q, moved, where = make(case, cuda_device, width=width)
    means = all_means(cache)
    got = flash_hog.paged_block_select(q.to(cuda_device), means.to(cuda_device), **where, page_size=16, blocks=20, first=2)
    assert torch.equal(got.cpu(), ref.select(q, means, cache.table, lengths, counts, 16, 20, 2, 1))


def test_select_beyond_the_table(cuda_device):
    """Tokens beyond the table have no list; those before them in the same tile have theirs."""
    import flash_hog

    gen = torch.Generator().manual_seed(0)
    means, q = torch.randn((20, 1, 64), generator=gen), torch.randn((40, 1, 64), generator=gen).to(BF16)
    table = torch.arange(20, dtype=torch.int32)[None]
    for length in (321, 330, 340, 2 ** 31 - 1):
        got = flash_hog.paged_block_select(
            q.to(cuda_device), means.to(cuda_device), table.to(cuda_device), torch.tensor([length], dtype=torch.int32, device=cuda_device),
            torch.tensor([0, 40], dtype=torch.int32, device=cuda_device), page_size=16, blocks=5)
        assert torch.equal(got.cpu(), ref.select(q, means, table, [length], [40], 16, 5, 1, 1)), length


@pytest.mark.parametrize("pages", [40, 300, 3000])
def test_ties_and_special_scores(pages, cuda_device):
    """Equal means tie, and ties go to the lowest column; signed zeros are equal; infinities are numbers, NaN is none."""
    print("[case] ties", pages, flush=True)
    gen = torch.Generator().manual_seed(pages)
    means = torch.randn((pages, 1, 64), generator=gen)
    q = torch.randn((1, 2, 64), generator=gen).to(BF16)
    length = 16 * pages - 3
    for kind in ("all", "some", "zeros", "special"):
        m = means.clone()
        if kind == "all":
            m[:] = m[0]
        elif kind == "some":
            m = m[torch.randint(0, 5, (pages,), generator=gen)]
        elif kind == "zeros":
            m[:] = 0
            m[1::2] = -0.0
        else:
            m[3], m[7], m[pages // 2], m[pages - 5] = float("nan"), float("inf"), float("-inf"), float("nan")
            m[11] = 0
            m[11, 0, 0] = float("inf") if q[0, :, 0].sum() > 0 else float("-inf")  # (0 * inf is no part of it)
        table = torch.arange(pages, dtype=torch.int32)[None]
        if kind == "special":
            table[0, 5], table[0, 6] = -1, pages
        for blocks in (1, 2, 5, 17, pages // 2, pages - 2):
            want = ref.select(q, m, table, [length], [1], 16, blocks, 0, 1)[0]
            for tiles in (False, True):
                got = choose(m, q, 16, blocks, length, cuda_device, table=table, tiles=tiles)
                assert torch.equal(got, want), (kind, blocks, tiles)


def test_close_scores(cuda_device):
    """Scores that fp32 cannot tell apart: a mean of 1 + k 2^-23 in one column against sums near 2^12."""
    print("[case] close scores", flush=True)
    gen = torch.Generator().manual_seed(0)
    pages = 200
    order = torch.randperm(pages, generator=gen)
    means = torch.full((pages, 1, 64), 64.0)
    means[:, 0, 17] = 1 + order * 2.0 ** -23
    q = torch.ones((1, 1, 64), dtype=BF16)
    want = torch.tensor(sorted([*order[:-1].argsort(descending=True)[:20].tolist(), pages - 1]), dtype=torch.int32)
    for tiles in (False, True):
        assert torch.equal(choose(means, q, 16, 21, 16 * pages, cuda_device, tiles=tiles)[0], want)


def test_rows_of_no_sequence(cuda_device):
    """A padded batch: lists of -1, rows of zeros, or as they were in an out that is given."""
    import flash_hog

    case = (4, 2, 64, BF16, False, 16, [100, 50], [3, 2], 4, 1, 1)
    cache, counts, q, moved, where = make(case, cuda_device)
    pad = torch.cat([q[:1], q, q[:2]]).to(cuda_device)
    where["query_offsets"] += 1
    means = all_means(cache).to(cuda_device)
    chosen = flash_hog.paged_block_select(pad, means, **where, page_size=16, blocks=4)
    want = ref.select(q, means.cpu(), cache.table, cache.lengths, counts, 16, 4, 1, 1)
    assert torch.equal(chosen[1:6].cpu(), want) and (chosen[[0, 6, 7]] == -1).all()
    chosen[[0, 6, 7]] = 0
    args = (pad, chosen, moved["key_cache"], moved["value_cache"])
    exact = ref.attention(q, cache, counts, want, 0.125)
    out = flash_hog.paged_block_attention(*args, **where)
    check(out[1:6], exact)
    assert not out[[0, 6, 7]].any()
    given = torch.full_like(pad, 7.0)
    version = given._version
    assert flash_hog.paged_block_attention(*args, **where, out=given) is given and given._version > version
    assert torch.equal(given[1:6], out[1:6]) and (given[[0, 6, 7]] == 7).all()


def test_bad_pages_and_lengths(cuda_device):
    """A chosen page outside the cache, or a length beyond the table, gives NaN in rows of its sequence only; offsets
    that fall or leave the rows stay inside them."""
    import flash_hog

    print("[case] bad pages", flush=True)
    case = (4, 2, 64, BF16, False, 16, [100, 100, 100], None, 3, 1, 1)
    cache, counts, q, moved, where = make(case, cuda_device)
    chosen = torch.tensor([[0, 2, 6]] * 6, dtype=torch.int32).view(3, 2, 3)
    args = (q.to(cuda_device), chosen.to(cuda_device), moved["key_cache"], moved["value_cache"])
    clean = flash_hog.paged_block_attention(*args, **where)
    for entry in (-1, cache.cache["k"].shape[0], 2 ** 31 - 1, -2 ** 31):
        table = moved["page_table"].clone()
        table[1, 2] = entry
        out = flash_hog.paged_block_attention(*args, **{**where, "page_table": table})
        assert torch.isnan(out[1]).all() and torch.equal(out[[0, 2]], clean[[0, 2]])
        table[1, 2], table[1, 3] = moved["page_table"][1, 2], entry  # not chosen
        assert torch.equal(flash_hog.paged_block_attention(*args, **{**where, "page_table": table}), clean)
    lengths = moved["lengths"].clone()
    lengths[2] = 2 ** 31 - 1
    out = flash_hog.paged_block_attention(*args, **{**where, "lengths": lengths})
    assert torch.isnan(out[2]).all() and torch.equal(out[:2], clean[:2])
    means = torch.randn((cache.cache["k"].shape[0], 2, 64), device=cuda_device)
    kept = means.clone()
    lists = flash_hog.paged_block_select(args[0], means, moved["page_table"], lengths, page_size=16, blocks=3)
    assert (lists[2] == -1).all() and (lists[:2, :, 2] == 6).all()
    flash_hog.paged_key_means(moved["key_cache"], means, moved["page_table"], lengths)
    assert torch.equal(means, kept)  # (length 100 fills no page, and the other is beyond its table)
    for offsets in ([0, 3, 2, 3], [5, 5, 5, 9], [-4, 1, 2, 2 ** 31 - 1], [2, 1, 0, -1]):
        more = {**where, "query_offsets": torch.tensor(offsets, dtype=torch.int32, device=cuda_device)}
        flash_hog.paged_key_means(moved["key_cache"], means, **more)
        lists = flash_hog.paged_block_select(args[0], means, **more, page_size=16, blocks=3)
        assert ((lists >= -1) & (lists < 8)).all()
        assert flash_hog.paged_block_attention(*args, **more).shape == q.shape


# (heads, kv_heads, head_dim, dtype, quantised, page, lengths, new, blocks): so many entries that blocks are taken
# one at a time
MANY = [
    (4, 4, 64, BF16, False, 64, [2000, 130, 0, 77], [400, 130, 0, 9], 13),
    (8, 4, 128, BF16, False, 128, [1500, 700], [333, 260], 8),
    (3, 3, 64, FP16, True, 64, [900, 1030], [260, 900], 15),
    (4, 2, 256, FP16, True, 128, [1700], [401], 9),
    (6, 2, 128, BF16, False, 256, [3000, 1, 300], [700, 1, 250], 7),
    (8, 8, 64, FP16, False, 16, [1300, 40], [1300, 40], 14),
    (2, 2, 256, BF16, False, 32, [2050], [2050], 17),
    (8, 2, 128, BF16, True, 64, [1200] * 5, [130, 64, 63, 1, 1200], 16),
    (32, 1, 64, BF16, False, 1024, [5000], [700], 4),             # 4 tokens a tile
    (5, 5, 128, BF16, False, 64, [8000], [300], 70),
    # a token at a time again: more blocks than a join's weights, more heads a group than a tile's rows
    (4, 2, 64, FP16, False, 16, [9000], [200], 300),
    (130, 1, 64, BF16, False, 256, [2000, 700], [500, 30], 3),
]


def many_lists(case, cache, counts, kind):
    """Rising lists as a choice gives them, or any: not rising, with columns twice, behind the token or outside the table."""
    blocks, T, N, width = case[8], sum(counts), case[1], cache.table.shape[1]
    gen = torch.Generator().manual_seed(4)
    if kind == "any":
        lists = torch.randint(-1, width + 2, (T, N, blocks), generator=gen).to(torch.int32)
        lists[::3, 0] = -1
        lists[1::4, :, min(3, blocks - 1)] = 2 ** 31 - 1
        lists[2::4, :, 2] = -2 ** 31
        return lists
    at = torch.cat([torch.arange(n - c, n) for n, c in zip(cache.lengths, counts)])
    own = (at // cache.page).clamp(min=0)[:, None, None]
    scores = torch.rand((T, N, width), generator=gen)
    columns = torch.arange(width)
    scores = torch.where(columns < own, scores, torch.where(columns == own, 2.0, -1.0))
    best, lists = scores.topk(min(blocks, width), -1)
    lists = torch.where(best >= 0, lists, 2 ** 31 - 1).sort(-1).values
    lists = torch.where(lists == 2 ** 31 - 1, -1, lists).to(torch.int32)
    return torch.nn.functional.pad(lists, (0, blocks - lists.shape[-1]), value=-1)


@pytest.mark.parametrize("kind", ["chosen", "any"])
@pytest.mark.parametrize("case", MANY, ids=lambda c: case_id((*c, 1, 1)))
def test_many_tokens(case, kind, cuda_device):
    import flash_hog

    print("[case] many tokens", case_id((*case, 1, 1)), kind, flush=True)
    cache, counts, q, moved, where = make(case, cuda_device)
    lists = many_lists(case, cache, counts, kind)
    for scale in (None, -0.21):
        got = flash_hog.paged_block_attention(q.to(cuda_device), lists.to(cuda_device), moved["key_cache"],
                                              moved["value_cache"], **where, **scales(moved), scale=scale)
        check(got, ref.attention_dense(q, cache, counts, lists, scale or q.shape[-1] ** -0.5), case_id((*case, 1, 1)))
    if kind == "any":
        assert not got[::3, :case[0] // case[1]].any()


def test_many_tokens_of_no_sequence(cuda_device):
    """Rows of no sequence between many that have one; pages outside the cache; lengths beyond the table and shorter
    than the new tokens; two sequences' tokens in one group of 64; offsets that fall, where all rows are NaN."""
    import flash_hog

    print("[case] many tokens of no sequence", flush=True)
    case = MANY[0]
    cache, counts, q, moved, where = make(case, cuda_device)
    lists = many_lists(case, cache, counts, "chosen")
    kv = moved["key_cache"], moved["value_cache"]
    pad = lambda x, value: torch.cat([torch.full_like(x[:70], value), x, torch.full_like(x[:33], value)])
    padded, plists = pad(q, 3.0).to(cuda_device), pad(lists, 0).to(cuda_device)
    more = {**where, "query_offsets": where["query_offsets"] + 70}
    exact = ref.attention_dense(q, cache, counts, lists, 0.125)
    out = flash_hog.paged_block_attention(padded, plists, *kv, **more)
    check(out[70:-33], exact)
    assert not out[:70].any() and not out[-33:].any()
    given = torch.full_like(padded, 7.0)
    assert flash_hog.paged_block_attention(padded, plists, *kv, **more, out=given) is given
    assert torch.equal(given[70:-33], out[70:-33]) and (given[:70] == 7).all() and (given[-33:] == 7).all()
    for entry in (-1, cache.cache["k"].shape[0], 2 ** 31 - 1, -2 ** 31):
        table = moved["page_table"].clone()
        table[0, 5] = entry
        hit = (lists == 5).any(-1) & (torch.arange(539) < 400)[:, None]
        bad = flash_hog.paged_block_attention(padded, plists, *kv, **{**more, "page_table": table})[70:-33]
        nan = torch.isnan(bad).all(-1).cpu()
        assert torch.equal(nan, hit) and torch.equal(torch.isnan(bad).any(-1).cpu(), hit)
        assert torch.equal(bad[~nan.to(cuda_device)], out[70:-33][~nan.to(cuda_device)])
    lengths = moved["lengths"].clone()
    lengths[1] = 2 ** 31 - 1
    bad = flash_hog.paged_block_attention(padded, plists, *kv, **{**more, "lengths": lengths})[70:-33]
    assert torch.isnan(bad[400:530]).all() and torch.equal(bad[:400], out[70:470]) and torch.equal(bad[530:], out[600:-33])
    lengths[1] = 100  # its first 30 tokens see nothing
    bad = flash_hog.paged_block_attention(padded, plists, *kv, **{**more, "lengths": lengths})[70:-33]
    assert not bad[400:430].any() and torch.equal(bad[:400], out[70:470]) and torch.equal(bad[530:], out[600:-33])
    rows = padded.shape[0]
    for offsets in ([0, 400, 300, 500, 600], [0, rows, 0, rows, rows], [rows, 300, 200, 100, 0], [-7, 60, 60, 70, 2 ** 31 - 1]):
        more["query_offsets"] = torch.tensor(offsets, dtype=torch.int32, device=cuda_device)
        out = flash_hog.paged_block_attention(padded, plists, *kv, **more)
        assert torch.isnan(out).all() if offsets[0] != -7 else torch.isfinite(out).all()
        # (lists of any values then, which the attention takes)
        choice = flash_hog.paged_block_select(padded, all_means(cache).to(cuda_device), **more, page_size=64, blocks=13)
        out = flash_hog.paged_block_attention(padded, choice, *kv, **more)
        assert torch.isnan(out).all() if offsets[0] != -7 else torch.isfinite(out).all()


def test_many_tokens_wide_table(cuda_device):
    """A table wider than a workgroup's masks, and one just as wide."""
    import flash_hog

    print("[case] many tokens, wide table", flush=True)
    case = MANY[6]
    for width in (None, 8192, 8193):
        cache, counts, q, moved, where = make(case, cuda_device, width=width)
        lists = many_lists(case, cache, counts, "chosen")
        out = flash_hog.paged_block_attention(q.to(cuda_device), lists.to(cuda_device), moved["key_cache"], moved["value_cache"], **where)
        check(out, ref.attention_dense(q, cache, counts, lists, 256 ** -0.5))


def test_strided_inputs(cuda_device):
    """Views: queries of a joint projection, lists and tables that are parts of wider ones."""
    import flash_hog

    for case in (CASES[8], CASES[13], (*MANY[0], 1, 1)):
        print("[case] strided", case_id(case), flush=True)
        cache, counts, q, moved, where = make(case, cuda_device)
        lists = many_lists(case, cache, counts, "chosen").to(cuda_device)
        q, means = q.to(cuda_device), all_means(cache).to(cuda_device)
        kv = moved["key_cache"], moved["value_cache"]
        wide = lambda t, axis: torch.cat([t, t.flip(0)], axis).narrow(axis, 0, t.shape[axis])
        strange = {**where, "page_table": wide(where["page_table"], 1), "lengths": torch.stack([where["lengths"]] * 2, 1)[:, 0]}
        if where["query_offsets"] is not None:
            strange["query_offsets"] = torch.stack([where["query_offsets"]] * 3, 1)[:, 1]
        assert not strange["page_table"].is_contiguous() or cache.table.shape[0] == 1
        out = flash_hog.paged_block_attention(q, lists, *kv, **where, **scales(moved))
        got = flash_hog.paged_block_attention(wide(q, 1), wide(lists, 2), *kv, **strange, **scales(moved))
        assert torch.equal(out, got)
        choice = [flash_hog.paged_block_select(x, means, **w, page_size=cache.page, blocks=4) for x, w in ((q, where), (wide(q, 2), strange))]
        assert torch.equal(*choice)


def test_two_streams(cuda_device):
    """Calls of two streams at once, each with workspaces of its own."""
    import flash_hog

    print("[case] two streams", flush=True)
    calls = []
    for case, kind in ((MANY[1], "chosen"), (MANY[7], "any"), (CASES[3], None)):
        cache, counts, q, moved, where = make(case, cuda_device)
        lists = many_lists(case, cache, counts, kind) if kind else ref.select(q, all_means(cache), cache.table, cache.lengths, counts, cache.page, *case[8:])
        q, lists, means = q.to(cuda_device), lists.to(cuda_device), all_means(cache).to(cuda_device)

        def call(q=q, lists=lists, means=means, moved=moved, where=where, page=cache.page):
            return (flash_hog.paged_block_attention(q, lists, moved["key_cache"], moved["value_cache"], **where, **scales(moved)),
                    flash_hog.paged_block_select(q, means, **where, page_size=page, blocks=5))
        calls.append(call)
    want = [call() for call in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    runs = []
    for _ in range(10):
        for stream, call in zip(streams, calls):
            with torch.cuda.stream(stream):
                runs.append(call())
    torch.cuda.synchronize()
    for i, run in enumerate(runs):
        assert all(torch.equal(a, b) for a, b in zip(run, want[i % len(calls)]))


def test_many_tokens_in_slabs(cuda_device):
    """More tokens than one slab holds, captured, replayed with other lists, and each like the call of its own."""
    import flash_hog

    print("[case] many tokens in slabs", flush=True)
    case = (8, 4, 64, BF16, False, 64, [6000, 5000], [5001, 4900], 64)  # 132 KiB a token and 1 GiB a slab
    cache, counts, q, moved, where = make(case, cuda_device)
    kv = moved["key_cache"], moved["value_cache"]
    q = q.to(cuda_device)
    runs = [many_lists(case, cache, counts, kind) for kind in ("chosen", "any")]
    want = [flash_hog.paged_block_attention(q, lists.to(cuda_device), *kv, **where) for lists in runs]
    check(want[1], ref.attention_dense(q.cpu(), cache, counts, runs[1], 0.125))
    given = runs[0].to(cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = flash_hog.paged_block_attention(q, given, *kv, **where)
    for i in (0, 1, 0, 1):
        given.copy_(runs[i])
        graph.replay()
        flash_hog.paged_block_attention(q, runs[1 - i].to(cuda_device), *kv, **where)
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])


def test_serving_loop(cuda_device):
    """What a server does at each step, captured and replayed: rows fork, grow by a token, norms and rotation, the
    token's key and value into the cache, means, choice, attention. Against the same in 64 bits, and, with
    all blocks chosen, against paged_attention."""
    import flash_hog
    import rotary_reference

    print("[case] serving loop", flush=True)
    B, H, N, D, page, pages, width, blocks = 4, 8, 2, 64, 16, 64, 12, 4
    gen = torch.Generator().manual_seed(12)
    dev = cuda_device
    k_cache, v_cache = (torch.full((pages, N, page, D), float("nan"), dtype=BF16, device=dev) for _ in "kv")
    means = torch.full((pages, N, D), float("nan"), device=dev)
    table = torch.full((B, width), -1, dtype=torch.int32, device=dev)
    lengths = torch.zeros(B, dtype=torch.int32, device=dev)
    freq = (10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)).float().to(dev)
    wq, wk = (torch.rand(D, generator=gen).to(BF16).to(dev) + 0.5 for _ in range(2))
    parents = torch.arange(B, dtype=torch.int32, device=dev)
    q, k, v = (torch.zeros((B, n, D), dtype=BF16, device=dev) for n in (H, N, N))

    def step(q, k, v, offsets, new):
        free = flash_hog.paged_cache_extend(k_cache, v_cache, table, lengths, new, parents)
        qr, kr = flash_hog.qk_norm_rotary(q, k, frequencies=freq, query_weight=wq, key_weight=wk, lengths=lengths,
                                          query_offsets=offsets)
        flash_hog.paged_cache_write(kr, v, k_cache, v_cache, table, lengths, offsets)
        flash_hog.paged_key_means(k_cache, means, table, lengths, offsets)
        chosen = flash_hog.paged_block_select(qr, means, table, lengths, offsets, page_size=page, blocks=blocks)
        return qr, kr, chosen, flash_hog.paged_block_attention(qr, chosen, k_cache, v_cache, table, lengths, offsets), free

    # a prompt of 70 tokens in row 0; then all rows go on from it
    rand = lambda n, heads: torch.randn((n, heads, D), generator=gen).to(BF16).to(dev)
    prompt = rand(70, H), rand(70, N), rand(70, N)
    offsets = torch.tensor([0, 70, 70, 70, 70], dtype=torch.int32, device=dev)
    new = torch.tensor([70, 0, 0, 0], dtype=torch.int32, device=dev)
    _, kr, _, _, free = step(*prompt, offsets, new)
    assert int(free) == pages - 5 and lengths.tolist() == [70, 0, 0, 0]
    history = [[(kr[i], prompt[2][i]) for i in range(70)], [], [], []]
    side = torch.cuda.Stream()
    saved = [t.clone() for t in (k_cache, v_cache, means, table, lengths)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(q, k, v, None, 1)
    torch.cuda.current_stream().wait_stream(side)
    for t, s in zip((k_cache, v_cache, means, table, lengths), saved):
        t.copy_(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qr, kr, chosen, out, free = step(q, k, v, None, 1)
    plans = [[0, 0, 0, 0], None, None, [0, 1, 1, 1], None, [2, 2, -1, 3]] + [None] * 20
    for plan in plans:
        parents.copy_(torch.tensor(plan or list(range(B)), dtype=torch.int32))
        history = [list(history[p]) if 0 <= p < B else [] for p in (plan or range(B))]
        for t, n in ((q, H), (k, N), (v, N)):
            t.copy_(rand(B, n))
        graph.replay()
        torch.cuda.synchronize()
        for b in range(B):
            history[b].append((kr[b].clone(), v[b].clone()))
        assert lengths.tolist() == [len(h) for h in history]
        assert int(free) == pages - len({x for row in table.tolist() for x in row if x >= 0})
        for b in range(B):
            n = len(history[b])
            keys, values = (torch.stack([h[i] for h in history[b]]).double().cpu() for i in range(2))
            want = rotary_reference.apply(q[b:b + 1].double().cpu(), wq.double().cpu(), torch.tensor([n - 1]), freq.cpu(), False, 1e-6)
            assert float((qr[b].double().cpu() - want[0]).abs().max()) <= 2.0 ** -8 * float(want.abs().max()) * 1.01
            full = (keys[:n // page * page].view(-1, page, N, D).sum(1) / page).float().double()
            for g in range(N):
                own = (n - 1) // page
                scores = full[:, g] @ qr[b, g * 4:(g + 1) * 4].double().cpu().sum(0)
                best = [0, own] if own else [0]
                for c in sorted(range(1, max(1, own)), key=lambda c: (-float(scores[c]), c)):
                    if len(best) < blocks:
                        best.append(c)
                best = sorted(best)
                assert chosen[b, g].tolist() == best + [-1] * (blocks - len(best))
                s = [c * page + r for c in best for r in range(page) if c * page + r < n]
                for h in range(g * 4, g * 4 + 4):
                    w = torch.softmax(keys[s, g] @ qr[b, h].double().cpu() * D ** -0.5, 0)
                    y = w @ values[s, g]
                    assert float((out[b, h].double().cpu() - y).abs().max()) <= 4 * 2.0 ** -8 * float(y.abs().max())


def test_far_offsets(cuda_device):
    """Pages and means beyond 2^32 bytes."""
    import flash_hog

    print("[case] far offsets", flush=True)
    pages, page, heads, dim = 9000, 16, 128, 256  # 1 MiB a page and tensor, 128 KiB of means
    k = torch.zeros((pages, heads, page, dim), dtype=BF16, device=cuda_device)
    v = torch.zeros_like(k)
    gen = torch.Generator().manual_seed(0)
    rows = torch.randn((2, 2, heads, page, dim), generator=gen).to(BF16)
    for i, at in enumerate((pages - 1, pages - 2)):
        k[at], v[at] = rows[0, i].to(cuda_device), rows[1, i].to(cuda_device)
    means = torch.zeros((40000, heads, dim), device=cuda_device)  # 5.2 GB
    means[39990] = 1.0
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=cuda_device)
    lengths = torch.tensor([32], dtype=torch.int32, device=cuda_device)
    mine = torch.zeros((pages, heads, dim), device=cuda_device)
    flash_hog.paged_key_means(k, mine, table, lengths)
    assert torch.equal(mine[pages - 2].cpu(), (rows[0, 1].double().sum(1) / 16).float()) and not mine[:pages - 2].any()
    q = torch.randn((1, heads, dim), generator=gen).abs().to(BF16)
    columns = torch.tensor([[5, 39990, 7, 8]], dtype=torch.int32, device=cuda_device)
    lists = flash_hog.paged_block_select(q.to(cuda_device), means, columns, lengths * 2, page_size=16, blocks=2, first=0)
    assert lists[0].tolist() == [[1, 3]] * heads
    out = flash_hog.paged_block_attention(q.to(cuda_device), torch.tensor([[[0, 1]] * heads], dtype=torch.int32, device=cuda_device),
                                          k, v, table, lengths)
    keys, values = (torch.cat([rows[n, 0], rows[n, 1]], 1).double() for n in range(2))
    w = torch.softmax((keys @ q[0].double()[:, :, None])[..., 0] * dim ** -0.5, -1)
    check(out[0], (w[:, None] @ values)[:, 0])


def test_slabs(cuda_device):
    """More scores than one slab holds: the choices of 300 tokens of 40000 pages are those of each alone."""
    import flash_hog

    print("[case] slabs", flush=True)
    gen = torch.Generator().manual_seed(0)
    means = torch.randn((40000, 4, 64), generator=gen).to(cuda_device)
    q = torch.randn((300, 4, 64), generator=gen).to(BF16).to(cuda_device)
    table = torch.randperm(40000, generator=gen).to(torch.int32)[None].to(cuda_device)
    lengths = torch.tensor([16 * 40000], dtype=torch.int32, device=cuda_device)
    offsets = torch.tensor([0, 300], dtype=torch.int32, device=cuda_device)
    got = flash_hog.paged_block_select(q, means, table, lengths, offsets, page_size=16, blocks=12)
    for i in (0, 150, 199, 208, 209, 210, 299):
        one = flash_hog.paged_block_select(q[i:i + 1], means, table, lengths - 299 + i, page_size=16, blocks=12)
        assert torch.equal(got[i:i + 1], one)
    scores = means[table[0].long(), 0].double() @ q[299, 0].double()
    scores[0] = scores[-1] = float("inf")
    assert got[299, 0].tolist() == sorted(scores.topk(12).indices.tolist())


@pytest.mark.parametrize("extension", [True, False])
def test_refusals(extension, cuda_device, monkeypatch):
    import flash_hog
    from flash_hog import _hip

    if not extension:
        monkeypatch.setattr(_hip, "torch_ext", lambda: None)
    case = CASES[1]
    cache, counts, q, moved, where = make(case, cuda_device)
    q = q.to(cuda_device)
    means = all_means(cache).to(cuda_device)
    chosen = torch.zeros((q.shape[0], 2, 4), dtype=torch.int32, device=cuda_device)
    kv = (moved["key_cache"], moved["value_cache"])
    select = lambda *a, **k: flash_hog.paged_block_select(*(a or (q, means)), **where, **{"page_size": 16, "blocks": 4, **k})
    attend = lambda *a, **k: flash_hog.paged_block_attention(*(a or (q, chosen)), *kv, **{**where, **k})
    for bad, error, match in (
            (lambda: select(q, means.half()), ValueError, "key_means has dtype"),
            (lambda: select(q, means[..., :32]), ValueError, "expected .* key_means"),
            (lambda: select(q, means[:, :, None].expand(-1, -1, 1, -1)), ValueError, "expected .* key_means"),
            (lambda: select(q[0], means), ValueError, r"expected a \(T, N, H\) query"),
            (lambda: select(q, means.transpose(0, 1).contiguous().transpose(0, 1)), ValueError, "contiguous"),
            (lambda: select(blocks=0), ValueError, "blocks must be 1 to 32768"),
            (lambda: select(blocks=32769), ValueError, "blocks must be 1 to 32768"),
            (lambda: select(first=4), ValueError, r"first \+ last <= blocks"),
            (lambda: select(last=0), ValueError, "last >= 1"),
            (lambda: select(first=-1), ValueError, "first >= 0"),
            (lambda: select(page_size=24), RuntimeError, "power of two"),
            (lambda: attend(q, chosen.long()), ValueError, "blocks must be torch.int32"),
            (lambda: attend(q, chosen[1:]), ValueError, "blocks must be torch.int32"),
            (lambda: attend(q, chosen[:, :1]), ValueError, "blocks must be torch.int32"),
            (lambda: attend(q, chosen[..., :0]), RuntimeError, "blocks must be >= 1"),
            (lambda: attend(scale=0.0), RuntimeError, "scale must be nonzero"),
            (lambda: attend(out=q), ValueError, "out overlaps query"),
            (lambda: attend(out=q[:, ::2].repeat(1, 2, 1).transpose(0, 1).contiguous().transpose(0, 1)), ValueError, "out must be contiguous"),
            (lambda: attend(lengths=moved["lengths"][:-1]), ValueError, "lengths has shape"),
            (lambda: flash_hog.paged_key_means(kv[0], means[:-1], **where), ValueError, "key_means has shape"),
            (lambda: flash_hog.paged_key_means(kv[0], means, **where, key_scale=chosen), ValueError, "e4m3 cache")):
        with pytest.raises(error, match=match):
            bad()
    grad = q.clone().requires_grad_()
    for bad in (lambda: select(grad, means), lambda: attend(grad, chosen), lambda: flash_hog.paged_key_means(kv[0], means.requires_grad_(), **where)):
        with pytest.raises(RuntimeError, match="has no derivative"):
            bad()


def test_repeats(cuda_device, monkeypatch):
    """The same bits at every call, with and without a table wider than needed, through the extension and without."""
    import flash_hog
    from flash_hog import _hip

    case = (8, 2, 128, BF16, True, 64, [6000, 2000], [40, 9], 12, 1, 2)
    for width in (None, 3000):
        cache, counts, q, moved, where = make(case, cuda_device, width=width)
        q, means = q.to(cuda_device), all_means(cache).to(cuda_device)
        runs = []
        for _ in range(2):
            chosen = flash_hog.paged_block_select(q, means, **where, page_size=64, blocks=12, last=2)
            runs.append((chosen, flash_hog.paged_block_attention(q, chosen, moved["key_cache"], moved["value_cache"], **where,
                                                                 **scales(moved))))
        assert all(torch.equal(a, b) for a, b in zip(*runs))
        if width is None:
            narrow = runs[0]
            monkeypatch.setattr(_hip, "torch_ext", lambda: None)
    assert all(torch.equal(a, b) for a, b in zip(narrow, runs[0]))
