"""The paged cache in use: captured and replayed decoding, streams, repeated calls, caches beyond
32-bit offsets, every value and every scale that a cache can hold, and random batches.

Tolerances: those of test_gpu_paged.py (check). Values written, quantised and read are compared
bit for bit.
"""

from __future__ import annotations

import pytest
import torch

import paged_reference as ref
from test_gpu_paged import CASES, case_id, check, make

pytestmark = pytest.mark.gpu

BF16, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def same(a, b):
    """Equal, NaN where the other is."""
    a, b = a.double().cpu(), b.double().cpu()
    return torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a, posinf=1e300, neginf=-1e300),
                                                                       torch.nan_to_num(b, posinf=1e300, neginf=-1e300))


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
def test_every_value_is_quantised(dtype, cuda_device):
    """All 65536 bit patterns as rows of 64 values, neighbours and at random."""
    import flash_hog

    print("[case] every value", dtype, flush=True)
    bits = torch.arange(65536, dtype=torch.int32)
    mixed = bits[torch.randperm(65536, generator=torch.Generator().manual_seed(0))]
    for values in (bits, mixed):
        x = values.to(torch.int16).view(dtype).view(1024, 1, 64)
        cache = [torch.zeros((64, 1, 16, 64), dtype=E4M3, device=cuda_device) for _ in range(2)]
        scale = [torch.zeros((64, 1, 16), dtype=torch.uint8, device=cuda_device) for _ in range(2)]
        kwargs = dict(page_table=torch.arange(64, dtype=torch.int32, device=cuda_device)[None],
                      lengths=torch.tensor([1024], dtype=torch.int32, device=cuda_device), key_scale=scale[0],
                      value_scale=scale[1])
        offsets = torch.tensor([0, 1024], dtype=torch.int32, device=cuda_device)
        flash_hog.paged_cache_write(x.to(cuda_device), x.flip(0).to(cuda_device), *cache, **kwargs,
                                    query_offsets=offsets)
        for c, s, rows in ((cache[0], scale[0], x), (cache[1], scale[1], x.flip(0))):
            codes, scales = ref.quantise(rows[:, 0])
            assert torch.equal(s.cpu().view(-1), scales)
            assert same(c.view(-1, 64).float(), codes.view(E4M3).float())


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
def test_every_scale_is_read(dtype, cuda_device):
    """All 256 e8m0 scales (255: NaN) with all 256 codes, to the nearest value of dtype; products
    below its normal range are as close as its smallest normal number."""
    import flash_hog

    print("[case] every scale", dtype, flush=True)
    codes = torch.arange(256, dtype=torch.uint8).view(1, 4, 64).expand(256, 4, 64).contiguous()  # (scale, part, column)
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1).expand(256, 4).contiguous()
    pages = codes.view(64, 1, 16, 64).to(cuda_device).view(E4M3)
    scale = scales.view(64, 1, 16).to(cuda_device)
    k, v = flash_hog.paged_cache_read(
        pages, pages, torch.arange(64, dtype=torch.int32, device=cuda_device)[None],
        torch.tensor([1024], dtype=torch.int32, device=cuda_device), dtype=dtype, key_scale=scale, value_scale=scale)
    assert same(k, v)
    assert torch.isnan(k.view(256, 4, 64)[255]).all()
    got = k.view(256, 4, 64)[:255].cpu()
    exact = codes[:255].view(E4M3).double() * ref.powers(scales[:255])[..., None]
    want = exact.to(dtype)  # (double to fp16 and bf16 rounds once)
    info = torch.finfo(dtype)
    normal = ~(exact.abs() < info.tiny) & ~torch.isnan(exact)
    assert torch.equal(got[normal], want[normal])
    assert torch.equal(torch.isnan(got), torch.isnan(exact))
    small = exact.abs() < info.tiny
    assert ((got[small].double() - exact[small]).abs() <= info.tiny).all()


def test_random_batches(cuda_device):
    """Heads, pages, lengths, new tokens, windows and sinks drawn at random."""
    import flash_hog

    gen = torch.Generator().manual_seed(17)
    draw = lambda *options: options[int(torch.randint(len(options), (1,), generator=gen))]
    number = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=gen))
    for i in range(40):
        Hk, batch = draw(1, 2, 3), number(1, 6)
        most = draw(20, 200, 1200)
        lengths = [number(0, most) for _ in range(batch)]
        new = None if draw(0, 1) else [number(0, min(n, 90)) for n in lengths]
        if new is not None and sum(new) == 0:
            new[0], lengths[0] = 1, max(lengths[0], 1)
        window = draw(0, 0, number(1, 300))
        case = (Hk * draw(1, 2, 4, 5, 9), Hk, draw(64, 128, 256), draw(BF16, FP16), draw(False, True), draw(16, 32, 64),
                lengths, new, window, draw(0, number(0, 100)) if window else 0)
        print("[case] random", i, case_id(case), flush=True)
        cache, counts, q, kwargs = make(case, cuda_device, seed=300 + i, width=draw(None, 300))
        out = flash_hog.paged_attention(q.to(cuda_device), **kwargs)
        want = ref.attention(q, cache, counts, case[8], case[9], q.shape[-1] ** -0.5)
        if want.abs().max() == 0:
            assert (out == 0).all()
        else:
            check(out, want, case_id(case))


def test_rows_before_the_first_sequence(cuda_device):
    import flash_hog

    print("[case] rows of no sequence", flush=True)
    for case in (CASES[14], CASES[16]):
        cache, counts, q, kwargs = make(case, cuda_device)
        want = flash_hog.paged_attention(q.to(cuda_device), **kwargs)
        padded = torch.cat([q[:2], q, q[:3]]).to(cuda_device)
        kwargs["query_offsets"] = kwargs["query_offsets"] + 2
        junk = torch.full_like(padded, float("nan"))  # (freed: what a fresh output may be made of)
        del junk
        got = flash_hog.paged_attention(padded, **kwargs)
        assert (got[:2] == 0).all() and (got[-3:] == 0).all()
        check(got[2:-3], ref.attention(q, cache, counts, case[8], case[9], q.shape[-1] ** -0.5))
        out = torch.full_like(padded, 3.0)
        flash_hog.paged_attention(padded, **kwargs, out=out)
        assert (out[:2] == 3).all() and (out[-3:] == 3).all() and torch.equal(out[2:-3], got[2:-3])
        assert want.shape == q.shape


@pytest.mark.parametrize("case", [CASES[7], CASES[16], (32, 8, 128, BF16, False, 16, [9000, 77], None, 0, 0)],
                         ids=["tokens", "chunk", "splits"])
def test_repeats_and_streams(case, cuda_device):
    """Repeated calls, and calls at once on two streams, give the same bits."""
    import flash_hog

    print("[case] repeats", case_id(case), flush=True)
    made = [make(case, cuda_device, seed=s) for s in (1, 2)]
    qs = [q.to(cuda_device) for _, _, q, _ in made]
    want = [flash_hog.paged_attention(q, **kwargs) for q, (_, _, _, kwargs) in zip(qs, made)]
    for (cache, counts, q, _), out in zip(made, want):
        check(out, ref.attention(q, cache, counts, case[8], case[9], q.shape[-1] ** -0.5))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    for _ in range(4):
        got = []
        for q, (_, _, _, kwargs), stream in zip(qs, made, streams):
            with torch.cuda.stream(stream):
                got.append(flash_hog.paged_attention(q, **kwargs))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_same_page_twice_and_strided_queries(cuda_device):
    """Sequences that share pages (a common prefix), one that names a page twice, and queries and
    index tensors that are not contiguous."""
    import flash_hog

    print("[case] shared pages", flush=True)
    cache = ref.Cache([64, 64, 64], 16, 2, 64, BF16, False, seed=3)
    cache.table[1, :2] = cache.table[0, :2]
    cache.table[2, 1] = cache.table[2, 0]
    kwargs = cache.on(cuda_device)
    q = torch.randn((3, 4, 64), generator=torch.Generator().manual_seed(1)).to(BF16)
    want = ref.attention(q, cache, [1, 1, 1], 0, 0, 0.125)
    check(flash_hog.paged_attention(q.to(cuda_device), **kwargs), want)
    wide = torch.zeros((3, 4, 128), dtype=BF16, device=cuda_device)
    wide[..., ::2] = q.to(cuda_device)
    kwargs["page_table"] = kwargs["page_table"].repeat_interleave(2, 1)[:, ::2]
    kwargs["lengths"] = kwargs["lengths"].repeat_interleave(2)[::2]
    check(flash_hog.paged_attention(wide[..., ::2], **kwargs), want)
    k, v = flash_hog.paged_cache_read(**kwargs, max_length=64)
    assert torch.equal(k[0, :32], k[1, :32]) and torch.equal(v[2, :16], v[2, 16:32])


@pytest.mark.parametrize("quantised", [False, True], ids=["plain", "e4m3"])
def test_decoding_graph_replays(quantised, cuda_device):
    """A decoding step (lengths advance, keys written, attention, a read) captured once and replayed
    for one token after another, with eager work between: the bits of eager steps."""
    import flash_hog

    print("[case] graph", quantised, flush=True)
    B, H, Hk, D, page, width = 3, 8, 2, 64, 16, 40
    gen = torch.Generator(device=cuda_device).manual_seed(2)
    kind = E4M3 if quantised else BF16

    def state():
        s = {"key_cache": torch.zeros((B * width, Hk, page, D), dtype=kind, device=cuda_device),
             "value_cache": torch.zeros((B * width, Hk, page, D), dtype=kind, device=cuda_device),
             "page_table": torch.randperm(B * width, generator=torch.Generator().manual_seed(5)).to(torch.int32)
             .view(B, width).to(cuda_device),
             "lengths": torch.tensor([0, 15, 300], dtype=torch.int32, device=cuda_device)}
        if quantised:
            s["key_scale"], s["value_scale"] = (torch.zeros((B * width, Hk, page), dtype=torch.uint8, device=cuda_device)
                                                for _ in range(2))
        return s

    def step(s, q, k, v):
        s["lengths"] += 1
        flash_hog.paged_cache_write(k, v, **s)
        out = flash_hog.paged_attention(q, **s, window=100, sinks=3)
        return out, *flash_hog.paged_cache_read(**s, max_length=64)

    q = torch.zeros((B, H, D), dtype=BF16, device=cuda_device)
    k, v = (torch.zeros((B, Hk, D), dtype=BF16, device=cuda_device) for _ in range(2))
    captured, eager = state(), state()
    start = {n: t.clone() for n, t in captured.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(captured, q, k, v)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outputs = step(captured, q, k, v)
    for n in captured:
        captured[n].view(torch.uint8).copy_(start[n].view(torch.uint8))
    torch.cuda.synchronize()
    for _ in range(6):
        for t in (q, k, v):
            t.normal_(generator=gen)
        want = step(eager, q.clone(), k.clone(), v.clone())
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outputs, want))
        assert torch.equal(captured["lengths"], eager["lengths"])


@pytest.mark.parametrize("quantised", [False, True], ids=["plain", "e4m3"])
def test_cache_beyond_32_bit_offsets(quantised, cuda_device):
    """Pages beyond 2^32 bytes (and 2^31 elements) of a cache: written, attended and read."""
    import flash_hog

    D, Hk, page = 256, 8, 64
    pages = (1 << 32) // (Hk * page * D) + 40  # of one-byte rows; twice that in bf16
    print("[case] large cache", pages, flush=True)
    kind = E4M3 if quantised else BF16
    kwargs = {n: torch.empty((pages, Hk, page, D), dtype=kind, device=cuda_device) for n in ("key_cache", "value_cache")}
    if quantised:
        for n in ("key_scale", "value_scale"):
            kwargs[n] = torch.empty((pages, Hk, page), dtype=torch.uint8, device=cuda_device)
    kwargs["page_table"] = torch.tensor([[pages - 1, 0, pages - 9, pages // 2 + 3]], dtype=torch.int32, device=cuda_device)
    N = 230
    kwargs["lengths"] = torch.tensor([N], dtype=torch.int32, device=cuda_device)
    offsets = torch.tensor([0, N], dtype=torch.int32, device=cuda_device)
    gen = torch.Generator(device=cuda_device).manual_seed(4)
    q, k, v = (torch.randn((N, n, D), generator=gen, device=cuda_device).to(BF16) for n in (2 * Hk, Hk, Hk))
    flash_hog.paged_cache_write(k, v, query_offsets=offsets, **kwargs)
    kd, vd = flash_hog.paged_cache_read(**kwargs, max_length=N)
    if not quantised:
        assert torch.equal(kd[0], k) and torch.equal(vd[0], v)
    got = flash_hog.paged_attention(q, query_offsets=offsets, **kwargs)
    last = flash_hog.paged_attention(q[-1:], **kwargs)
    scores = (q.double().transpose(0, 1) @ kd[0].double().repeat_interleave(2, 1).permute(1, 2, 0)) * D ** -0.5
    scores = scores.masked_fill(torch.ones(N, N, dtype=torch.bool, device=cuda_device).triu(1), float("-inf"))
    want = (torch.softmax(scores, -1) @ vd[0].double().repeat_interleave(2, 1).transpose(0, 1)).transpose(0, 1)
    check(got, want.cpu())
    check(last, want[-1:].cpu())


def test_long_read_beyond_32_bit_offsets(cuda_device):
    """A read of more than 2^31 elements, through a table that names a few pages over and over."""
    import flash_hog

    Hk, D, page = 8, 128, 64
    width = (1 << 31) // (page * Hk * D) + 3
    print("[case] long read", width, flush=True)
    cache = torch.randn((5, Hk, page, D), device=cuda_device).to(BF16)
    table = (torch.arange(width, dtype=torch.int32, device=cuda_device) % 5)[None]
    length = torch.tensor([width * page - 7], dtype=torch.int32, device=cuda_device)
    k, v = flash_hog.paged_cache_read(cache, -cache, table, length)
    assert k.numel() > 1 << 31
    for p in (0, width // 2, width - 2):
        assert torch.equal(k[0, p * page:(p + 1) * page], cache[p % 5].transpose(0, 1))
    assert torch.equal(v[0, -page:-7], -cache[(width - 1) % 5].transpose(0, 1)[:-7])
    assert (k[0, -7:] == 0).all() and (v[0, -7:] == 0).all()


def test_refused_calls_on_the_device(cuda_device, monkeypatch):
    """Shapes, types and layouts that do not fit: the same error from both wrappers, nothing launched."""
    import flash_hog
    from flash_hog import _hip

    print("[case] refusals", flush=True)
    cache = ref.Cache([20, 3], 16, 2, 64, BF16, False)
    x = cache.on(cuda_device)
    eight = ref.Cache([20, 3], 16, 2, 64, BF16, True).on(cuda_device)
    q, k = (torch.zeros((2, n, 64), dtype=BF16, device=cuda_device) for n in (4, 2))
    a, w, r = flash_hog.paged_attention, flash_hog.paged_cache_write, flash_hog.paged_cache_read
    without = lambda d, *names: {n: t for n, t in d.items() if n not in names}
    calls = [
        (lambda: a(q[0], **x), "expected a \\(T, N, H\\) query"),
        (lambda: a(q.half(), **x), "the cache must be of"),
        (lambda: a(q.float(), **{**x, "key_cache": x["key_cache"].float(), "value_cache": x["value_cache"].float()}), "dtype"),
        (lambda: a(q[..., :32], **x), "disagree on head_dim"),
        (lambda: a(q[:, :3], **x), "multiple of kv_heads"),
        (lambda: a(q[:1], **x), "one row a sequence"),
        (lambda: a(q, **x, out=torch.empty_like(q[:1])), "out has shape"),
        (lambda: a(q, **x, out=torch.empty_like(q.half())), "dtype"),
        (lambda: a(q, **x, out=torch.empty((2, 4, 128), dtype=BF16, device=cuda_device)[..., ::2]), "out must be contiguous"),
        (lambda: a(q, **{**x, "key_cache": x["key_cache"].transpose(1, 2)}), "value_cache has shape|contiguous"),
        (lambda: a(q, **{**x, "lengths": x["lengths"].long()}), "expected torch.int32"),
        (lambda: a(q, **{**x, "page_table": x["page_table"][0]}), "page_table"),
        (lambda: a(q, **{**x, "lengths": x["lengths"][:1]}), "lengths has shape"),
        (lambda: a(q, **x, query_offsets=x["lengths"]), "query_offsets has shape"),
        (lambda: a(q, **without(eight, "key_scale")), "an e4m3 cache needs key_scale"),
        (lambda: a(q, **x, key_scale=eight["key_scale"], value_scale=eight["value_scale"]), "are for an e4m3 cache"),
        (lambda: a(q, **{**eight, "key_scale": eight["key_scale"].view(torch.int8)}), "float8_e8m0fnu or torch.uint8"),
        (lambda: a(q, **{**x, "value_cache": x["value_cache"].cpu()}), "must be on a GPU device"),
        (lambda: w(k, k[..., :32], **x), "value has shape"),
        (lambda: w(k, k.half(), **x), "dtype"),
        (lambda: w(q, q, **x), "disagree on heads or head_dim"),
        (lambda: r(**x, dtype=FP16), "the cache must be of"),
        (lambda: r(**x, max_length=-1), "max_length must be >= 0"),
        (lambda: r(**{**x, "key_cache": x["key_cache"][:, :, :8].contiguous(),
                      "value_cache": x["value_cache"][:, :, :8].contiguous()}), "page_size must be a power of two"),
    ]
    for python in (False, True):
        if python:
            monkeypatch.setattr(_hip, "torch_ext", lambda: None)
        for i, (call, needle) in enumerate(calls):
            with pytest.raises((ValueError, TypeError, _hip.FlashHogError), match=needle):
                call()
                pytest.fail(f"call {i} was accepted")


@pytest.mark.parametrize("D,dtype,new,kv_heads", [(64, BF16, 260, 192), (64, FP16, 64, 256), (128, FP16, 260, 192),
                                                   (128, BF16, 64, 256), (256, BF16, 260, 192)])
def test_long_chunks(D, dtype, new, kv_heads, cuda_device):
    """Chunks that sweep thousands of keys in one go (heads enough that no split is made), in tiles
    of 128 rows and of 64; then with a page far back that is none."""
    import flash_hog

    length, page = 9000, 32
    print("[case] long chunk", D, dtype, new, kv_heads, flush=True)
    gen = torch.Generator(device=cuda_device).manual_seed(D + new)
    pages = -(-length // page)
    cache = [torch.randn((pages, kv_heads, page, D), generator=gen, device=cuda_device, dtype=dtype) for _ in "kv"]
    table = torch.randperm(pages, generator=gen, device=cuda_device).to(torch.int32)[None]
    q = torch.randn((new, kv_heads, D), generator=gen, device=cuda_device, dtype=dtype)
    kwargs = dict(lengths=torch.tensor([length], dtype=torch.int32, device=cuda_device),
                  query_offsets=torch.tensor([0, new], dtype=torch.int32, device=cuda_device))
    out = flash_hog.paged_attention(q, *cache, table, **kwargs)
    hidden = torch.ones((new, length), dtype=torch.bool, device=cuda_device).triu(length - new + 1)
    for head in (0, kv_heads // 2 + 1, kv_heads - 1):
        k, v = (c[table[0].long(), head].flatten(0, 1)[:length].double() for c in cache)
        scores = (q[:, head].double() @ k.T * D ** -0.5).masked_fill(hidden, float("-inf"))
        check(out[:, head], (torch.softmax(scores, -1) @ v).cpu(), str(head))
    table[0, pages - 3] = -1  # most tiles lie before it; tokens at positions from its first key on see it
    out = flash_hog.paged_attention(q, *cache, table, **kwargs)
    first = max(0, page * (pages - 3) - (length - new))
    assert bool(torch.isnan(out[first:]).all())


@pytest.mark.parametrize("batch", [2, 63, 64, 65])
@pytest.mark.parametrize("quantised", [False, True], ids=["plain", "e4m3"])
def test_sorted_tiles(batch, quantised, cuda_device):
    """Chunks whose tiles are taken longest first (up to 64 sequences) and by sequence (65): empty
    ones among them, equal lengths, fewer keys than new tokens, several tiles with the same keys."""
    import flash_hog

    print("[case] sorted", batch, quantised, flush=True)
    new = [(0, 1, 150, 40, 40, 3)[i % 6] + (i % 7 == 3) for i in range(batch)]
    lengths = [max(n - 2, 0) if i % 5 == 4 else n + 30 * (i % 3) for i, n in enumerate(new)]
    lengths[-1], new[-1] = 200, 170
    for heads, kv_heads, head_dim in ((2, 2, 64), (200, 1, 64), (6, 2, 128)):
        if heads == 200 and batch > 2:
            continue
        case = (heads, kv_heads, head_dim, BF16, quantised, 16, lengths, new, 0, 0)
        cache, counts, q, kwargs = make(case, cuda_device, seed=batch)
        out = flash_hog.paged_attention(q.to(cuda_device), **kwargs)
        check(out, ref.attention(q, cache, counts, 0, 0, q.shape[-1] ** -0.5), str(batch))
