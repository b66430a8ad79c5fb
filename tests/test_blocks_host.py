"""Attention over chosen blocks without a GPU: refusals of the C ABI and the front-end, shapes on fake tensors,
and the rules that split work."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import flash_hog
from flash_hog import _hip

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def lib():
    return _hip.lib()


def means_args(ptr=16, scale=None, means=16, table=16, offsets=None, batch=3, kv_heads=2, head_dim=64, num_pages=4,
               page_size=16, width=5, cache=2):
    return [None, ptr, scale, means, table, table, offsets, batch, kv_heads, head_dim, num_pages, page_size, width, cache]


def select_args(ptr=16, means=16, table=16, offsets=None, chosen=16, ws=16, size=1 << 40, batch=3, total=3, heads=4, kv_heads=2,
                head_dim=64, num_pages=4, page_size=16, width=5, dtype=2, blocks=4, first=1, last=1):
    return [None, ptr, means, table, table, offsets, chosen, ws, size, batch, total, heads, kv_heads, head_dim, num_pages,
            page_size, width, dtype, blocks, first, last]


def attention_args(ptr=16, chosen=16, scale_ptr=None, table=16, offsets=None, out=16, ws=16, size=1 << 40, batch=3, total=3,
                   heads=4, kv_heads=2, head_dim=64, num_pages=4, page_size=16, width=5, dtype=2, cache=2, blocks=4, scale=0.125):
    return [None, ptr, chosen, ptr, ptr, scale_ptr, scale_ptr, table, table, offsets, out, ws, size, batch, total, heads, kv_heads,
            head_dim, num_pages, page_size, width, dtype, cache, blocks, 1, scale]


SIZES = [(dict(batch=-1), 1, "sizes must not be negative"), (dict(kv_heads=0), 1, "sizes must be >= 1"),
         (dict(num_pages=0), 1, "sizes must be >= 1"), (dict(width=0), 1, "sizes must be >= 1"),
         (dict(page_size=17), 1, "power of two"), (dict(head_dim=80), 2, "head_dim must be 64, 128 or 256"),
         (dict(width=1 << 28), 1, "problem too large"), (dict(offsets=6), 1, "query_offsets is not 4-byte aligned"),
         (dict(ptr=None), 1, "null"), (dict(ptr=8), 1, "not 16-byte aligned"), (dict(table=None), 1, "page_table is null")]
TOKENS = [(dict(total=4), 1, "without query_offsets there is one row a sequence"), (dict(heads=3), 1, "multiple of kv_heads"),
          (dict(dtype=0), 2, "dtype must be bf16 or fp16"), (dict(blocks=0), 1, "blocks must be >= 1"),
          (dict(blocks=40000), 2, "blocks must be <= 32768"), (dict(chosen=None), 1, "chosen is null"),
          (dict(batch=0, total=2, offsets=16), 1, "rows without a sequence"), (dict(total=-1), 1, "sizes must not be negative")]


@pytest.mark.parametrize("kwargs,status,needle", SIZES + [
    (dict(cache=0), 2, "dtype must be"), (dict(cache=3), 1, "needs k_scale"), (dict(means=None), 1, "key_means is null"),
    (dict(means=6), 1, "not 4-byte aligned")])
def test_means_refusals(lib, kwargs, status, needle):
    assert lib.fhog_paged_key_means(*means_args(**kwargs)) == status
    assert needle in lib.fhog_last_error().decode()


@pytest.mark.parametrize("kwargs,status,needle", SIZES + TOKENS + [
    (dict(first=-1), 1, "first >= 0"), (dict(last=0), 1, "last >= 1"), (dict(first=3, last=2), 1, "first + last <= blocks"),
    (dict(first=(1 << 31) - 1, last=2), 1, "first + last <= blocks"), (dict(ws=None, width=2000), 1, "workspace is null"),
    (dict(size=100, width=2000), 1, "below its"), (dict(ws=4, width=2000), 1, "8-byte aligned"), (dict(means=8), 1, "not 16-byte aligned"),
    (dict(width=(1 << 21) + 1), 1, "problem too large")])
def test_select_refusals(lib, kwargs, status, needle):
    assert lib.fhog_paged_block_select(*select_args(**kwargs)) == status
    assert needle in lib.fhog_last_error().decode()


@pytest.mark.parametrize("kwargs,status,needle", SIZES + TOKENS + [
    (dict(scale=0.0), 2, "nonzero"), (dict(scale=float("nan")), 1, "finite"), (dict(cache=1), 2, "the cache must be of"),
    (dict(cache=3), 1, "needs k_scale"), (dict(out=None), 1, "out is null"), (dict(blocks=1 << 14, page_size=1 << 17, width=1), 2, "2^30 keys"),
    (dict(total=1 << 22, batch=1 << 22), 1, "problem too large"), (dict(ws=None, blocks=256, page_size=64), 1, "workspace is null")])
def test_attention_refusals(lib, kwargs, status, needle):
    assert lib.fhog_paged_block_attention(*attention_args(**kwargs)) == status
    assert needle in lib.fhog_last_error().decode()


def test_nothing_to_do(lib):
    assert lib.fhog_paged_key_means(*means_args(batch=0, ptr=None, table=None)) == 0
    assert lib.fhog_paged_block_select(*select_args(batch=0, total=0, ptr=None, table=None, chosen=None, ws=None, size=0)) == 0
    assert lib.fhog_paged_block_attention(*attention_args(batch=0, total=0, ptr=None, table=None, chosen=None)) == 0


def test_workspace_bytes(lib):
    """Scores of the tokens of a slab: all of them, or as many as 256 MiB hold; at least one. None where LDS holds
    them."""
    scores = lambda *sizes: lib.fhog_paged_block_select_workspace_bytes(*sizes, 1, 1)
    assert scores(10, 10, 1, 4, 64, 2000) == 10 * 4 * 2000 * 8
    assert scores(1, 7, 0, 4, 64, 2000) == 7 * 4 * 2000 * 8
    assert scores(10, 10, 1, 4, 128, 1026) == 0 and scores(10, 10, 1, 4, 256, 1026) == 10 * 4 * 1026 * 8  # a workgroup a token
    assert scores(512, 512, 1, 1, 64, 100) == 0 and scores(513, 513, 1, 1, 64, 100) == 513 * 100 * 8
    assert scores(1, 1000, 0, 4, 256, 1026) == 0 and scores(1, 1000, 0, 4, 256, 1027) == 1000 * 4 * 1027 * 8  # tiles
    assert scores(1, 1 << 20, 0, 8, 64, 2048) == 1 << 28
    assert scores(5, 5, 1, 64, 64, 1 << 21) == 64 * 8 << 21
    assert scores(0, 0, 1, 4, 64, 100) == 0
    assert lib.fhog_paged_block_workspace_bytes(1, 1, 1, 4, 2, 64, 16, 5, 1) == 0
    assert lib.fhog_paged_block_workspace_bytes(1, 1, 1, 4, 2, 64, 15, 5, 1) == 0
    few, many = (lib.fhog_paged_block_workspace_bytes(t, t, 1, 32, 8, 128, 64, 500, 64) for t in (1, 4096))
    assert few > 0 and many == 0
    # many tokens: their blocks' outputs, a slab of 1 GiB at a time; a token at a time where 64 tokens' do not fit
    outputs = lambda heads, dim, page, blocks, total=1 << 15: lib.fhog_paged_block_workspace_bytes(
        1, total, 0, heads, 8, dim, page, 512, blocks)
    assert 32 * 16 * 130 * 4 * 2035 < outputs(32, 128, 64, 16, 2035) < 32 * 16 * 130 * 4 * 2035 + (64 << 20)
    assert 0.9 * 2 ** 30 < outputs(32, 128, 64, 16) < 1.1 * 2 ** 30
    assert outputs(64, 256, 1024, 253) > 0 and outputs(64, 256, 1024, 255) == 0


def cpu(kind=BF16, device="cpu"):
    x = dict(key_cache=torch.zeros(4, 2, 16, 64, dtype=kind, device=device),
             value_cache=torch.zeros(4, 2, 16, 64, dtype=kind, device=device),
             page_table=torch.zeros(3, 2, dtype=torch.int32, device=device),
             lengths=torch.ones(3, dtype=torch.int32, device=device))
    if kind == E4M3:
        x.update({n: torch.zeros(4, 2, 16, dtype=torch.uint8, device=device) for n in ("key_scale", "value_scale")})
    return x


def calls(x, q, means, chosen):
    where = {n: x[n] for n in ("page_table", "lengths")}
    return (lambda: flash_hog.paged_key_means(x["key_cache"], means, **where, key_scale=x.get("key_scale")),
            lambda: flash_hog.paged_block_select(q, means, **where, page_size=16, blocks=2),
            lambda: flash_hog.paged_block_attention(q, chosen, **x))


def test_front_end_refuses():
    x, q = cpu(), torch.zeros(3, 4, 64, dtype=BF16)
    means, chosen = torch.zeros(4, 2, 64), torch.zeros(3, 2, 2, dtype=torch.int32)
    for call in calls(x, q, means, chosen):
        with pytest.raises(ValueError, match="must be on a GPU device"):
            call()
    with pytest.raises(TypeError):
        flash_hog.paged_block_select(q, means, x["page_table"], x["lengths"], page_size=16, blocks=2.5)
    for call in calls(x, q.float().requires_grad_(), means.requires_grad_(), chosen):
        with pytest.raises(RuntimeError, match="has no derivative"):
            call()
    for i, name in enumerate(("paged_key_means", "paged_block_select", "paged_block_attention")):
        with pytest.raises(RuntimeError, match="vmap"):
            torch.func.vmap(lambda n: calls({**x, "lengths": n}, q, means.detach(), chosen)[i]())(torch.ones(2, 3, dtype=torch.int32))


@pytest.mark.parametrize("kind", [BF16, E4M3], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("device", ["cuda", "cpu"])
def test_fake_tensors(device, kind):
    with FakeTensorMode():
        x, q = cpu(kind, device), torch.zeros(3, 4, 64, dtype=BF16, device=device)
        means = torch.zeros(4, 2, 64, device=device)
        chosen = torch.zeros(3, 2, 2, dtype=torch.int32, device=device)
        none, lists, out = (call() for call in calls(x, q, means, chosen))
        assert none is None and lists.shape == (3, 2, 2) and lists.dtype == torch.int32
        assert out.shape == q.shape and out.dtype == BF16 and out.device == q.device
        with pytest.raises(ValueError, match="out is not supported"):
            flash_hog.paged_block_attention(q, chosen, **x, out=torch.empty_like(q))


def test_workspace_of_long_lists(lib):
    """Lists of more blocks than a split holds have parts for every token, within 1 GiB for however many tokens."""
    size = lambda total, heads, kv_heads, dim, page, blocks: lib.fhog_paged_block_workspace_bytes(
        1, total, 0, heads, kv_heads, dim, page, 4096, blocks)
    for shape in ((4, 4, 64, 16, 600), (8, 8, 128, 16, 2000), (64, 1, 256, 64, 4096), (32, 8, 128, 32, 32768)):
        one, few, many = (size(total, *shape) for total in (1, 300, 60000))
        assert 0 < one and few <= many <= 1 << 30 and many > 0.9 * 2 ** 30
