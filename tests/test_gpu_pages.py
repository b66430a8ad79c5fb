"""paged_cache_extend and paged_cache_compact against their definition (pages_reference.py). Everything is
compared bit for bit: the allocator computes whole numbers and copies."""

from __future__ import annotations

import pytest
import torch

import pages_reference as ref

pytestmark = pytest.mark.gpu

BF16, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def cache(pages, heads, page, dim, kind, device, seed=0):
    """Random bytes, so that every copy shows."""
    gen = torch.Generator(device=device).manual_seed(seed)
    bits = lambda *s: torch.randint(0, 256, s, generator=gen, device=device, dtype=torch.uint8)
    item = 1 if kind == E4M3 else 2
    x = {n: bits(pages, heads, page, dim * item).view(kind) for n in ("key_cache", "value_cache")}
    if kind == E4M3:
        x.update({n: bits(pages, heads, page) for n in ("key_scale", "value_scale")})
    return x


def raw(t):
    return t.contiguous().view(torch.uint8).cpu()


def i32(x, device):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=device)


def check_extend(table, lengths, parents, new, pages, page, heads, dim, kind, device, each=None):
    import flash_hog

    x = cache(pages, heads, page, dim, kind, device)
    before = {n: raw(t) for n, t in x.items()}
    t, n = i32(table, device), i32(lengths, device)
    free = flash_hog.paged_cache_extend(x["key_cache"], x["value_cache"], t, n, i32(new, device) if each is None else each,
                                        i32(parents, device), **{k: v for k, v in x.items() if "scale" in k})
    want_table, want_lengths, want_free, copies = ref.extend(table, lengths, parents, new, pages, page)
    assert t.tolist() == want_table and n.tolist() == want_lengths
    assert free.shape == () and free.dtype == torch.int32 and int(free) == want_free
    for name, value in before.items():
        want = value.clone()
        for source, target, rows in copies:
            want[target, :, :rows] = value[source, :, :rows]
        assert torch.equal(raw(x[name]), want), name
    return copies


@pytest.mark.parametrize("kind", [BF16, FP16, E4M3], ids=["bf16", "fp16", "e4m3"])
@pytest.mark.parametrize("seed", range(8))
def test_extend(seed, kind, cuda_device):
    page, heads, dim = (16, 32, 64, 128)[seed % 4], (1, 2, 3)[seed % 3], (64, 128, 256)[seed % 3]
    pages = (40, 7, 200)[seed % 3]
    print("[case] extend", seed, kind, page, heads, dim, pages, flush=True)
    args = ref.scenario(seed, 13, 5, pages, page)
    check_extend(*args, pages, page, heads, dim, kind, cuda_device)


@pytest.mark.parametrize("batch,width,pages,page", [
    (1, 1, 1, 16), (2, 3, 5, 256), (1500, 3, 6000, 16), (64, 2048, 32768, 16), (70, 2000, 32768, 16), (70, 1800, 70000, 16),
    (20000, 2, 32769, 32), (3, 5, 40000, 64)])
def test_sizes(batch, width, pages, page, cuda_device):
    """More rows than threads, the most pages and entries that one workgroup books, and more than those."""
    print("[case] sizes", batch, width, pages, page, flush=True)
    args = ref.scenario(batch + pages, batch, width, pages, page)
    check_extend(*args, pages, page, 1, 64, E4M3, cuda_device)


def test_forks_part_ways(cuda_device):
    """One prompt, four rows: the first keeps the last page, the others get copies; a step later nobody shares it."""
    import flash_hog

    table, lengths = [[5, 2, -1], [-1] * 3, [-1] * 3, [-1] * 3], [20, 0, 0, 0]
    copies = check_extend(table, lengths, [0] * 4, [1] * 4, 8, 16, 2, 64, BF16, cuda_device, each=1)
    assert copies == [(2, 0, 4), (2, 1, 4), (2, 3, 4)]
    x = cache(8, 2, 16, 64, BF16, cuda_device)
    t, n = i32(table, cuda_device), i32(lengths, cuda_device)
    caches = (x["key_cache"], x["value_cache"])
    assert int(flash_hog.paged_cache_extend(*caches, t, n, 1, i32([0] * 4, cuda_device))) == 3
    assert t.tolist() == [[5, 2, -1], [5, 0, -1], [5, 1, -1], [5, 3, -1]] and n.tolist() == [21] * 4
    assert int(flash_hog.paged_cache_extend(*caches, t, n, 0)) == 3 and n.tolist() == [21] * 4
    # all but one end, and their pages are free at once
    n[1:] = 0
    assert int(flash_hog.paged_cache_extend(*caches, t, n, 0)) == 6
    # row 2 goes on from row 0, row 0 takes tokens back into the shared first page
    assert int(flash_hog.paged_cache_extend(*caches, t, n, 12, i32([0, -1, 0, -1], cuda_device))) == 1
    assert t.tolist() == [[5, 2, 0], [1, -1, -1], [5, 3, 4], [6, -1, -1]]
    n[0] = 3
    assert int(flash_hog.paged_cache_extend(*caches, t, n, i32([1, 0, 0, 0], cuda_device))) == 2
    assert t.tolist()[0] == [0, -1, -1] and n.tolist() == [4, 12, 33, 12]


def test_lacking_pages(cuda_device):
    copies = check_extend([[0, 1], [0, 1], [2, -1]], [20, 20, 16], None, [40, 1, 5], 4, 16, 1, 64, BF16, cuda_device)
    assert copies == [(1, 3, 4)]


@pytest.mark.parametrize("kind", [BF16, E4M3], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("seed", range(6))
def test_compact(seed, kind, cuda_device):
    import flash_hog

    batch, width, pages, page, heads, dim = [(13, 5, 40, 16, 2, 64), (1, 1, 1, 32, 1, 128), (40, 9, 300, 64, 8, 128),
                                             (9, 4, 50, 256, 3, 256), (300, 500, 1000, 16, 1, 64),
                                             (8, 3, 40000, 16, 1, 64)][seed]
    table, lengths, _, _ = ref.scenario(seed, batch, width, pages, page)
    x = cache(pages, heads, page, dim, kind, cuda_device)
    x["key_means"] = torch.randn((pages, heads, dim), device=cuda_device)
    for out_pages in (None, 1, pages + 3, 17):
        print("[case] compact", seed, kind, out_pages, flush=True)
        got = flash_hog.paged_cache_compact(x["key_cache"], x["value_cache"], i32(table, cuda_device),
                                            i32(lengths, cuda_device), num_pages=out_pages,
                                            **{k: v for k, v in x.items() if k[4:] != "cache" and k != "value_cache"})
        count = pages if out_pages is None else out_pages
        used, want_table = ref.compact(table, lengths, pages, page, count)
        assert got[5].tolist() == want_table
        used = used[:count]
        for name, y in zip(("key_cache", "value_cache", "key_scale", "value_scale", "key_means"), got):
            if name not in x:
                assert y is None
                continue
            assert y.shape == (count, *x[name].shape[1:]) and y.dtype == x[name].dtype
            assert torch.equal(raw(y)[:len(used)], raw(x[name])[used]), name
            assert not raw(y)[len(used):].any(), name


def test_compact_without_rows(cuda_device):
    import flash_hog

    x = cache(4, 2, 16, 64, BF16, cuda_device)
    got = flash_hog.paged_cache_compact(x["key_cache"], x["value_cache"], torch.empty((0, 3), dtype=torch.int32, device=cuda_device),
                                        torch.empty(0, dtype=torch.int32, device=cuda_device))
    assert got[5].shape == (0, 3) and not raw(got[0]).any() and got[2] is None


def test_far_offsets(cuda_device):
    """Pages beyond 2^32 bytes of a cache."""
    import flash_hog

    print("[case] far offsets", flush=True)
    pages, page, heads, dim = 1100, 256, 16, 256  # 2 MiB a page and tensor
    x = [torch.zeros((pages, heads, page, dim), dtype=BF16, device=cuda_device) for _ in range(2)]
    last = torch.randn((heads, page, dim), device=cuda_device).to(BF16)
    x[0][1099], x[1][1099] = last, -last
    x[0][1098, 0, 0, 0] = 3
    t, n = i32([[1099, -1], [1099, -1]] + [[i, i + 549] for i in range(549)], cuda_device), i32([100, 100] + [512] * 549, cuda_device)
    assert int(flash_hog.paged_cache_extend(*x, t, n, i32([1, 1] + [0] * 549, cuda_device))) == 0
    assert t[:2].tolist() == [[1099, -1], [1098, -1]]
    for c, want in zip(x, (last, -last)):
        assert torch.equal(c[1098, :, :100], want[:, :100]) and not c[1098, :, 100:].any()
    k, v, _, _, _, table = flash_hog.paged_cache_compact(*x, t, n)
    assert table[0, 0] == 1099 and torch.equal(k[1099], last) and torch.equal(v[1099], -last)


def test_graph_and_streams(cuda_device):
    """A captured step forks and grows anew at every replay, from tables and lengths that change in place; the
    same call on another stream."""
    import flash_hog

    print("[case] graph", flush=True)
    page, pages = 16, 60
    x = cache(pages, 2, page, 64, E4M3, cuda_device)
    args = (x["key_cache"], x["value_cache"])
    scales = {k: v for k, v in x.items() if "scale" in k}
    t, n = torch.full((6, 4), -1, dtype=torch.int32, device=cuda_device), torch.zeros(6, dtype=torch.int32, device=cuda_device)
    parents, new = i32(list(range(6)), cuda_device), i32([1] * 6, cuda_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        flash_hog.paged_cache_extend(*args, t, n, new, parents, **scales)
    torch.cuda.current_stream().wait_stream(side)
    assert n.tolist() == [1] * 6 and t[:, 0].tolist() == list(range(6))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        free = flash_hog.paged_cache_extend(*args, t, n, new, parents, **scales)
        moved = flash_hog.paged_cache_compact(*args, t, n, **scales)
    for seed in range(5):
        table, lengths, par, more = ref.scenario(seed, 6, 4, pages, page, wild=False)
        par = list(range(6)) if par is None else par
        for to, values in ((t, table), (n, lengths), (parents, par), (new, more)):
            to.copy_(i32(values, cuda_device))
        before = {k: raw(v) for k, v in x.items()}
        graph.replay()
        torch.cuda.synchronize()
        want, want_lengths, left, copies = ref.extend(table, lengths, par, more, pages, page)
        assert t.tolist() == want and n.tolist() == want_lengths and int(free) == left, seed
        for name, value in before.items():
            for source, target, rows in copies:
                value[target, :, :rows] = value[source, :, :rows]
            assert torch.equal(raw(x[name]), value)
        used, want = ref.compact(want, want_lengths, pages, page, pages)
        assert moved[5].tolist() == want and torch.equal(raw(moved[0])[:len(used)], raw(x["key_cache"])[used])


@pytest.mark.parametrize("extension", [True, False])
def test_versions_and_refusals(extension, cuda_device, monkeypatch):
    """Written tensors get a new autograd version; wrong arguments raise before anything is written."""
    import flash_hog
    from flash_hog import _hip

    if not extension:
        monkeypatch.setattr(_hip, "torch_ext", lambda: None)

    x = cache(4, 2, 16, 64, BF16, cuda_device)
    t, n = i32([[0, -1]], cuda_device), i32([3], cuda_device)
    args = (x["key_cache"], x["value_cache"])
    versions = [y._version for y in (*args, t, n)]
    flash_hog.paged_cache_extend(*args, t, n, 1)
    assert all(y._version > v for y, v in zip((*args, t, n), versions))
    with torch.inference_mode():
        flash_hog.paged_cache_extend(*args, t, n, 1)
    wide = i32([[0, -1, -1, -1]], cuda_device)[:, ::2]
    for bad, match in ((lambda: flash_hog.paged_cache_extend(*args, wide, n, 1), "page_table must be contiguous"),
                       (lambda: flash_hog.paged_cache_extend(*args, t, n, n), "new_tokens overlaps"),
                       (lambda: flash_hog.paged_cache_extend(*args, t, n, 1, n), "parents overlaps"),
                       (lambda: flash_hog.paged_cache_extend(*args, t, n, 1, i32([0, 0], cuda_device)), "parents has shape"),
                       (lambda: flash_hog.paged_cache_extend(*args, t, n, torch.ones(1, device=cuda_device)), "new_tokens has dtype"),
                       (lambda: flash_hog.paged_cache_extend(*args, t, n, -1), "new_tokens must be >= 0"),
                       (lambda: flash_hog.paged_cache_extend(*args, t[:0], n[:0], 1), "at least one row"),
                       (lambda: flash_hog.paged_cache_extend(*args, t, n, 1, torch.zeros(1, dtype=torch.int32)), "GPU device"),
                       (lambda: flash_hog.paged_cache_compact(*args, t, n, num_pages=0), "num_pages must be >= 1"),
                       (lambda: flash_hog.paged_cache_compact(*args, t, n, key_means=torch.zeros((4, 2, 64), dtype=BF16, device=cuda_device)),
                        "key_means has dtype"),
                       (lambda: flash_hog.paged_cache_compact(*args, t, n, key_scale=t), "are for an e4m3 cache")):
        with pytest.raises(ValueError, match=match):
            bad()
    assert n.tolist() == [5]


def test_compact_many_pages_without_rows(cuda_device):
    """More pages than one workgroup keeps books of, and no row: zeros."""
    import flash_hog

    print("[case] many pages without rows", flush=True)
    x = [torch.ones((40000, 1, 16, 64), dtype=BF16, device=cuda_device) for _ in range(2)]
    none = torch.empty((0, 3), dtype=torch.int32, device=cuda_device)
    got = flash_hog.paged_cache_compact(*x, none, none[:, 0], num_pages=33000)
    assert got[0].shape[0] == 33000 and not raw(got[0]).any() and not raw(got[1]).any() and got[5].shape == (0, 3)


def test_pages_of_two_gib(cuda_device):
    """A head of a page of 2^31 bytes: a fork's copy, and a compaction."""
    import flash_hog

    print("[case] pages of 2 GiB", flush=True)
    page = 1 << 22
    x = [torch.empty((3, 1, page, 256), dtype=BF16, device=cuda_device) for _ in range(2)]
    columns = torch.arange(256, device=cuda_device)
    for i, c in enumerate(x):
        c[2, 0] = ((torch.arange(page, device=cuda_device)[:, None] * (3 + i) + columns) % 251).to(BF16)
        c[0], c[1] = -1.0, -2.0
    t, n = i32([[2], [2]], cuda_device), i32([page - 5, page - 5], cuda_device)
    assert int(flash_hog.paged_cache_extend(*x, t, n, i32([1, 0], cuda_device))) == 1
    assert t.tolist() == [[0], [2]] and n.tolist() == [page - 4, page - 5]
    for c in x:
        assert torch.equal(c[0, 0, :-5], c[2, 0, :-5]) and (c[0, 0, -5:] == -1).all() and (c[1] == -2).all()
    k, v, _, _, _, table = flash_hog.paged_cache_compact(*x, t[1:].contiguous(), n[1:].contiguous(), num_pages=2)
    assert table.tolist() == [[0]]
    for got, c in ((k, x[0]), (v, x[1])):
        assert torch.equal(got[0], c[2]) and not got[1].any()
