"""Attention over a paged cache, writing and reading it, against plain 64-bit forms.

Tolerances, fixed before the first run, with u = eps / 2 of the output's type. Attention: the
output's own rounding and that of the probabilities that enter the value product, u each, and
the scores' fp32 error, which is far below: 2-norm of the error at most 2 u of the output's
(roundings of a row's terms average out), 4 u of the largest entry for a single one. e4m3 caches
are compared with the values they hold, which bf16 holds exactly and fp16 in these ranges.
Quantised codes, scales and what is read back are equal bit for bit.
"""

from __future__ import annotations

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def check(got, want, what=""):
    u = torch.finfo(got.dtype).eps / 2
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    norm, top = want.norm().item(), want.abs().max().item()
    err, big = (got - want).norm().item(), (got - want).abs().max().item()
    assert err <= 2 * u * norm, f"{what}: 2-norm error {err / max(norm, 1e-30):.2e} > {2 * u:.2e}"
    assert big <= 4 * u * top, f"{what}: largest error {big / max(top, 1e-30):.2e} > {4 * u:.2e}"


# (heads, kv_heads, head_dim, dtype, quantised, page, lengths, new (None: one each), window, sinks)
CASES = [
    (1, 1, 64, BF16, False, 16, [1], None, 0, 0),
    (4, 2, 64, BF16, False, 16, [1, 15, 16, 17, 0, 33, 200], None, 0, 0),
    (12, 4, 64, FP16, False, 16, [70, 331], None, 0, 0),
    (8, 1, 128, BF16, False, 32, [5, 500], None, 0, 0),
    (16, 1, 128, BF16, False, 64, [31, 32, 63], None, 0, 0),
    (34, 2, 64, BF16, False, 16, [40, 77], None, 0, 0),          # 17 heads a group
    (4, 4, 256, BF16, False, 16, [100, 257], None, 0, 0),
    (8, 2, 128, BF16, True, 64, [1, 64, 65, 1000], None, 0, 0),
    (8, 2, 64, FP16, True, 16, [3, 90, 700], None, 0, 0),
    (4, 2, 256, FP16, True, 128, [129, 300], None, 0, 0),
    (4, 2, 64, BF16, False, 16, [1, 40, 500], None, 24, 0),
    (4, 2, 64, BF16, False, 16, [1, 40, 500, 1500], None, 100, 5),
    (4, 2, 128, BF16, True, 32, [37, 900], None, 1, 1),
    (4, 2, 64, FP16, False, 16, [600], None, 33, 70),            # sinks beyond one tile
    (4, 2, 64, BF16, False, 16, [50, 3, 20], [7, 3, 1], 0, 0),
    (2, 2, 64, BF16, False, 16, [50, 3, 0, 200], [50, 2, 0, 33], 0, 0),
    (8, 2, 128, BF16, False, 16, [300, 80], [64, 80], 0, 0),
    (4, 1, 128, FP16, False, 64, [700], [129], 0, 0),
    (2, 1, 256, BF16, False, 16, [150, 90], [70, 20], 0, 0),
    (8, 2, 128, BF16, True, 64, [300, 80], [64, 80], 0, 0),
    (4, 2, 64, FP16, True, 16, [333, 40], [100, 40], 0, 0),
    (2, 1, 256, BF16, True, 32, [150], [70], 0, 0),
    (4, 2, 64, BF16, False, 16, [400, 80, 60], [150, 80, 1], 50, 4),
    (4, 2, 128, BF16, True, 16, [400, 30], [90, 3], 17, 40),
    (2, 2, 64, BF16, False, 16, [300], [300], 1, 0),             # a token sees itself alone
    (6, 2, 64, BF16, False, 16, [3, 2], [5, 2], 0, 0),           # more new tokens than the length: two see nothing
]


def case_id(c):
    H, Hk, D, dt, q8, page, lengths, new, w, s = c
    n = "x".join(map(str, lengths))
    return f"h{H}_{Hk}_d{D}_{str(dt)[6:]}{'_e4m3' if q8 else ''}_p{page}_len{n}" + \
        (f"_new{'x'.join(map(str, new))}" if new else "") + f"_w{w}_s{s}"


def make(c, device, seed=5, width=None):
    H, Hk, D, dtype, quantised, page, lengths, new, window, sinks = c
    cache = ref.Cache(lengths, page, Hk, D, dtype, quantised, seed=seed, width=width)
    counts = new or [1] * len(lengths)
    gen = torch.Generator().manual_seed(seed + 1)
    q = torch.randn((sum(counts), H, D), generator=gen).to(dtype)
    kwargs = cache.on(device)
    if new:
        offsets = torch.zeros(len(new) + 1, dtype=torch.int32)
        offsets[1:] = torch.cumsum(torch.tensor(new), 0)
        kwargs["query_offsets"] = offsets.to(device)
    kwargs.update(window=window or None, sinks=sinks)
    return cache, counts, q, kwargs


def run(c, device, **more):
    import flash_hog

    print("[case]", case_id(c), more, flush=True)
    cache, counts, q, kwargs = make(c, device, **{k: more.pop(k) for k in ("seed", "width") if k in more})
    scale = more.get("scale") or q.shape[-1] ** -0.5
    out = flash_hog.paged_attention(q.to(device), **kwargs, **more)
    check(out, ref.attention(q, cache, counts, c[8], c[9], scale), case_id(c))


@pytest.mark.parametrize("case", CASES, ids=case_id)
def test_attention(case, cuda_device):
    run(case, cuda_device)


@pytest.mark.parametrize("case", [CASES[3], CASES[8], CASES[17], CASES[22]], ids=case_id)
def test_attention_other_scales(case, cuda_device):
    run(case, cuda_device, scale=-0.21, seed=9)


@pytest.mark.parametrize("case", [CASES[1], CASES[7], CASES[11], CASES[14], CASES[19]], ids=case_id)
def test_attention_wide_table(case, cuda_device):
    """A table of many pages a sequence: as many splits of the keys, most of them empty."""
    run(case, cuda_device, width=2048)


@pytest.mark.parametrize("case", [CASES[1], CASES[8], CASES[16], CASES[20]], ids=case_id)
def test_python_wrappers_agree(case, cuda_device, monkeypatch):
    """FLASH_HOG_TORCH_EXT=0's wrappers give the extension's bits."""
    import flash_hog
    from flash_hog import _hip

    print("[case] wrappers", case_id(case), flush=True)
    _, _, q, kwargs = make(case, cuda_device)
    a = flash_hog.paged_attention(q.to(cuda_device), **kwargs)
    monkeypatch.setattr(_hip, "torch_ext", lambda: None)
    b = flash_hog.paged_attention(q.to(cuda_device), **kwargs)
    assert torch.equal(a, b)


@pytest.mark.parametrize("chunk", [False, True], ids=["tokens", "chunk"])
def test_rows_behind_the_last_sequence(chunk, cuda_device):
    """A padded batch: with out its padding stays, without it is zero."""
    import flash_hog

    print("[case] padding", chunk, flush=True)
    case = CASES[16] if chunk else CASES[14]
    cache, counts, q, kwargs = make(case, cuda_device)
    want = flash_hog.paged_attention(q.to(cuda_device), **kwargs)
    padded = torch.cat([q, torch.full_like(q[:3], float("nan"))]).to(cuda_device)
    out = torch.full_like(padded, 7.0)
    got = flash_hog.paged_attention(padded, **kwargs, out=out)
    assert got is out
    check(got[:-3], ref.attention(q, cache, counts, case[8], case[9], q.shape[-1] ** -0.5))
    assert (got[-3:] == 7.0).all()
    fresh = flash_hog.paged_attention(padded, **kwargs)
    assert torch.equal(fresh[:-3], got[:-3]) and (fresh[-3:] == 0).all()
    check(want, ref.attention(q, cache, counts, case[8], case[9], q.shape[-1] ** -0.5))


@pytest.mark.parametrize("case", [CASES[1], CASES[16]], ids=case_id)
def test_bad_pages_and_lengths(case, cuda_device):
    """What the host cannot check: the sequences concerned give NaN, the others their values."""
    import flash_hog

    print("[case] bad pages", case_id(case), flush=True)
    cache, counts, q, kwargs = make(case, cuda_device)
    want = ref.attention(q, cache, counts, case[8], case[9], q.shape[-1] ** -0.5)
    starts = [sum(counts[:b]) for b in range(len(counts) + 1)]
    last = len(counts) - 1
    rows = slice(starts[last], starts[last + 1])
    for bad in (-1, 1 << 30, kwargs["key_cache"].shape[0], "length"):
        broken = dict(kwargs)
        if bad == "length":
            broken["lengths"] = kwargs["lengths"].clone()
            broken["lengths"][last] = (1 << 31) - 1
        else:
            broken["page_table"] = kwargs["page_table"].clone()
            broken["page_table"][last, 0] = bad
        got = flash_hog.paged_attention(q.to(cuda_device), **broken)
        assert torch.isnan(got[rows]).all(), bad
        check(got[:rows.start], want[:rows.start], str(bad))


def test_offsets_out_of_range(cuda_device):
    """Offsets beyond the packed rows, or falling, are cut: whatever comes out, memory is safe."""
    import flash_hog

    print("[case] offsets", flush=True)
    for case in (CASES[14], CASES[16]):
        _, _, q, kwargs = make(case, cuda_device)
        n = kwargs["lengths"].numel()
        for offsets in ([-5] + [10**9] * n, [9] + [3] * n, [0] * n + [-1]):
            kwargs["query_offsets"] = torch.tensor(offsets, dtype=torch.int32, device=cuda_device)
            out = flash_hog.paged_attention(q.to(cuda_device), **kwargs)
            assert out.shape == q.shape
    torch.cuda.synchronize()


def test_freed_pages_before_the_window(cuda_device):
    """Pages that only hidden keys lie in may be gone from the table."""
    import flash_hog

    print("[case] freed pages", flush=True)
    for new, window, sinks in ((None, 40, 5), ([30], 40, 5), ([30], 40, 0)):
        case = (4, 2, 64, BF16, False, 16, [300], new, window, sinks)
        cache, counts, q, kwargs = make(case, cuda_device)
        want = ref.attention(q, cache, counts, window, sinks, q.shape[-1] ** -0.5)
        first = 300 - counts[0] - window + 1  # first key of the first token's window
        table = kwargs["page_table"]
        table[0, (1 if sinks else 0):first // 16] = -1
        check(flash_hog.paged_attention(q.to(cuda_device), **kwargs), want)


def test_empty_calls(cuda_device):
    import flash_hog

    cache = ref.Cache([5], 16, 2, 64, BF16, False)
    kwargs = cache.on(cuda_device)
    q = torch.empty((0, 4, 64), dtype=BF16, device=cuda_device)
    offsets = torch.zeros(2, dtype=torch.int32, device=cuda_device)
    assert flash_hog.paged_attention(q, **kwargs, query_offsets=offsets).shape == (0, 4, 64)
    flash_hog.paged_cache_write(q[:, :2], q[:, :2], **kwargs, query_offsets=offsets)
    k, v = flash_hog.paged_cache_read(**kwargs, max_length=0)
    assert k.shape == v.shape == (1, 0, 2, 64)
    # rows but no new tokens at all
    q = torch.ones((3, 4, 64), dtype=BF16, device=cuda_device)
    assert (flash_hog.paged_attention(q, **kwargs, query_offsets=offsets) == 0).all()


# ------------------------------------------------------------------ write and read

@pytest.mark.parametrize("quantised", [False, True], ids=["plain", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 64), (256, 32)])
def test_write_and_read(D, page, dtype, quantised, cuda_device):
    import flash_hog

    print("[case] write", D, page, dtype, quantised, flush=True)
    lengths, new = [1, 40, 0, 100, 33], [1, 17, 0, 100, 2]
    cache = ref.Cache(lengths, page, 3, D, dtype, quantised)
    kwargs = cache.on(cuda_device)
    total = sum(new) + 2  # two rows of padding
    gen = torch.Generator().manual_seed(3)
    k, v = (torch.randn((total, 3, D), generator=gen) * torch.exp(torch.randn((total, 3, 1), generator=gen))
            for _ in range(2))
    k[0, 0], k[1, 1] = 0.0, 448.0              # a row of zeros; magnitudes at a scale's edge
    k[2, 0, 3], k[3, 1, 5], k[4, 2, 0] = float("nan"), float("inf"), -float("inf")
    v[1, 0], v[2, 1], v[3, 0] = 449.0, 1e-7, 60000.0
    k, v = k.to(dtype), v.to(dtype)
    offsets = torch.zeros(len(new) + 1, dtype=torch.int32)
    offsets[1:] = torch.cumsum(torch.tensor(new), 0)
    flash_hog.paged_cache_write(k.to(cuda_device), v.to(cuda_device), **kwargs, query_offsets=offsets.to(cuda_device))

    want = {n: cache.cache[n].clone() for n in "kv"}
    scales = {n: cache.scale[n].clone() for n in "kv"} if quantised else None
    row = 0
    for b, (count, length) in enumerate(zip(new, lengths)):
        for i in range(count):
            p = length - count + i
            at = (int(cache.table[b, p // page]), slice(None), p % page)
            for n, x in (("k", k), ("v", v)):
                if quantised:
                    codes, scale = ref.quantise(x[row])
                    want[n].view(torch.uint8)[at], scales[n][at] = codes, scale
                else:
                    want[n][at] = x[row]
            row += 1
    for n, name in (("k", "key"), ("v", "value")):
        got = kwargs[name + "_cache"].cpu()
        if quantised:
            assert torch.equal(kwargs[name + "_scale"].cpu().view(torch.uint8), scales[n])
            a, b = got.float(), want[n].float()  # (a NaN's sign is free)
        else:
            a, b = got.float(), want[n].float()
        assert torch.equal(torch.isnan(a), torch.isnan(b))
        assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))
        cache.cache[n] = want[n]
        if quantised:
            cache.scale[n] = scales[n]

    read = flash_hog.paged_cache_read(**kwargs, max_length=90, dtype=dtype)
    for n, got in zip("kv", read):
        assert got.shape == (5, 90, 3, D) and got.dtype == dtype
        for b, length in enumerate(lengths):
            seen = min(length, 90)
            a, r = got[b, :seen].cpu(), cache.rows(n, b, length)[:seen].to(dtype)
            assert torch.equal(torch.isnan(a), torch.isnan(r))
            assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(r))
            assert (got[b, seen:] == 0).all()


def test_write_one_token_each(cuda_device):
    import flash_hog

    cache = ref.Cache([5, 0, 33], 16, 2, 64, BF16, False)
    kwargs = cache.on(cuda_device)
    before = kwargs["key_cache"].clone()
    k = torch.randn((3, 2, 64)).to(BF16).to(cuda_device)
    flash_hog.paged_cache_write(k, -k, **kwargs)
    for b, p in ((0, 4), (2, 32)):  # the empty sequence's row goes nowhere
        page = int(cache.table[b, p // 16])
        assert torch.equal(kwargs["key_cache"][page, :, p % 16], k[b])
        assert torch.equal(kwargs["value_cache"][page, :, p % 16], -k[b])
        before[page, :, p % 16] = k[b]
    assert torch.equal(before.view(torch.int16), kwargs["key_cache"].view(torch.int16))


def test_write_and_read_bad_pages(cuda_device):
    import flash_hog

    print("[case] write to bad pages", flush=True)
    cache = ref.Cache([20, 20], 16, 2, 64, BF16, False)
    kwargs = cache.on(cuda_device)
    before = kwargs["key_cache"].clone()
    kwargs["page_table"][0, 1] = 1 << 30
    kwargs["lengths"][1] = (1 << 31) - 1
    k = torch.randn((2, 2, 64)).to(BF16).to(cuda_device)
    flash_hog.paged_cache_write(k, k, **kwargs)
    assert torch.equal(before.view(torch.int16), kwargs["key_cache"].view(torch.int16))
    got, _ = flash_hog.paged_cache_read(**kwargs, max_length=64)
    assert torch.equal(got[0, :16].cpu().double(), cache.rows("k", 0, 16)) and torch.isnan(got[0, 16:20]).all()
    assert (got[0, 20:] == 0).all() and torch.isnan(got[1, 48:]).all()


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("quantised", [False, True], ids=["plain", "e4m3"])
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3)])
def test_prompt_and_tokens_match_the_dense_forward(window, sinks, quantised, cuda_device):
    """A sequence served in pieces (a prompt's chunks, then single tokens: write, then attend) gives
    what one dense causal call over its (cached) keys and values gives."""
    import flash_hog

    print("[case] together", window, sinks, quantised, flush=True)
    N, H, Hk, D, page = 203, 8, 2, 64, 16
    gen = torch.Generator().manual_seed(8)
    q, k, v = (torch.randn((N, n, D), generator=gen).to(BF16).to(cuda_device) for n in (H, Hk, Hk))
    kind = torch.float8_e4m3fn if quantised else BF16
    caches = [torch.zeros((20, Hk, page, D), dtype=kind, device=cuda_device) for _ in range(2)]
    kwargs = {"page_table": torch.randperm(20, generator=gen).to(torch.int32).to(cuda_device)[None],
              "key_cache": caches[0], "value_cache": caches[1]}
    if quantised:
        for n in ("key_scale", "value_scale"):
            kwargs[n] = torch.zeros((20, Hk, page), dtype=torch.uint8, device=cuda_device).view(torch.float8_e8m0fnu)
    got, at = [], 0
    for count in [100, 64, 30] + [1] * 9:
        lengths = torch.tensor([at + count], dtype=torch.int32, device=cuda_device)
        offsets = None if count == 1 else torch.tensor([0, count], dtype=torch.int32, device=cuda_device)
        piece = slice(at, at + count)
        flash_hog.paged_cache_write(k[piece], v[piece], lengths=lengths, query_offsets=offsets, **kwargs)
        got.append(flash_hog.paged_attention(q[piece], lengths=lengths, query_offsets=offsets, window=window,
                                             sinks=sinks, **kwargs))
        at += count
    kd, vd = flash_hog.paged_cache_read(lengths=lengths, max_length=N, dtype=BF16, **kwargs)
    if not quantised:
        assert torch.equal(kd[0], k) and torch.equal(vd[0], v)
    with torch.no_grad():
        want = flash_hog.dot_product_attention(q[None], kd, vd, is_causal=True, window=window, sinks=sinks)[0]
    # two implementations, each within the tolerance of the exact result
    got = torch.cat(got).double()
    u = torch.finfo(BF16).eps / 2
    assert (got - want.double()).norm() <= 2 * 2 * u * want.double().norm()
    assert (got - want.double()).abs().max() <= 2 * 4 * u * want.double().abs().max()
