"""The paged cache's allocator without a GPU: refusals of the C ABI and the front-end, shapes on fake
tensors, and the oracle's own invariants."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import flash_hog
import pages_reference as ref
from flash_hog import _hip

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def lib():
    return _hip.lib()


def extend_args(ptr=16, scales=16, table=16, free=16, parents=None, new=None, each=1, ws=16, size=1 << 30, batch=3, kv_heads=2,
                head_dim=64, num_pages=4, page_size=16, width=5, cache=2):
    return [None, ptr, ptr, scales, scales, table, table, parents, new, each, free, ws, size, batch, kv_heads, head_dim,
            num_pages, page_size, width, cache]


def compact_args(ptr=16, scales=16, table=16, means=None, means_out=None, ws=16, size=1 << 30, batch=3, kv_heads=2, head_dim=64,
                 num_pages=4, page_size=16, width=5, out=4, cache=2):
    return [None, ptr, ptr, scales, scales, means, table, table, ptr, ptr, scales, scales, means_out, table, ws, size, batch,
            kv_heads, head_dim, num_pages, page_size, width, out, cache]


BOTH = [
    (dict(ptr=None), 1, "k_cache is null"),
    (dict(ptr=8), 1, "not 16-byte aligned"),
    (dict(table=None), 1, "page_table is null"),
    (dict(table=6), 1, "not 4-byte aligned"),
    (dict(ws=None), 1, "workspace is null"),
    (dict(size=16), 1, "below its"),
    (dict(batch=-1), 1, "sizes must not be negative"),
    (dict(kv_heads=0), 1, "sizes must be >= 1"),
    (dict(num_pages=0), 1, "sizes must be >= 1"),
    (dict(width=0), 1, "sizes must be >= 1"),
    (dict(page_size=24), 1, "power of two"),
    (dict(page_size=8), 1, "power of two"),
    (dict(head_dim=96), 2, "head_dim must be 64, 128 or 256"),
    (dict(cache=0), 2, "dtype must be bf16 or fp16"),
    (dict(cache=7), 2, "dtype must be bf16 or fp16"),
    (dict(batch=1 << 20, width=1 << 12), 1, "problem too large"),
    (dict(kv_heads=70000), 1, "problem too large"),
    (dict(cache=3, scales=None), 1, "scale"),
]


@pytest.mark.parametrize("kwargs,status,needle", BOTH + [
    (dict(free=None), 1, "free_pages is null"), (dict(each=-1), 1, "new_each must be >= 0"), (dict(batch=0), 1, "no rows"),
    (dict(parents=6), 1, "4-byte aligned"), (dict(new=6), 1, "4-byte aligned")])
def test_extend_refusals(lib, kwargs, status, needle):
    assert lib.fhog_paged_cache_extend(*extend_args(**kwargs)) == status
    assert needle in lib.fhog_last_error().decode()


@pytest.mark.parametrize("kwargs,status,needle", BOTH + [
    (dict(out=0), 1, "out_pages must be >= 1"), (dict(means=16), 1, "go together"), (dict(means=8, means_out=8), 1, "16-byte"),
    (dict(cache=3, scales=8), 1, "16-byte aligned")])
def test_compact_refusals(lib, kwargs, status, needle):
    assert lib.fhog_paged_cache_compact(*compact_args(**kwargs)) == status
    assert needle in lib.fhog_last_error().decode()


def cpu(kind=BF16, device="cpu"):
    x = dict(key_cache=torch.zeros(4, 2, 16, 64, dtype=kind, device=device),
             value_cache=torch.zeros(4, 2, 16, 64, dtype=kind, device=device),
             page_table=torch.zeros(3, 2, dtype=torch.int32, device=device),
             lengths=torch.ones(3, dtype=torch.int32, device=device))
    if kind == E4M3:
        x.update({n: torch.zeros(4, 2, 16, dtype=torch.uint8, device=device) for n in ("key_scale", "value_scale")})
    return x


def test_front_end_refuses():
    x = cpu()
    with pytest.raises(ValueError, match="must be on a GPU device"):
        flash_hog.paged_cache_extend(new_tokens=1, **x)
    with pytest.raises(ValueError, match="must be on a GPU device"):
        flash_hog.paged_cache_compact(**x)
    with pytest.raises(TypeError):
        flash_hog.paged_cache_extend(new_tokens=1.5, **x)
    grad = {**x, "key_cache": x["key_cache"].float().requires_grad_()}
    for call in (lambda: flash_hog.paged_cache_extend(new_tokens=1, **grad), lambda: flash_hog.paged_cache_compact(**grad)):
        with pytest.raises(RuntimeError, match="has no derivative"):
            call()
    with pytest.raises(RuntimeError, match="vmap"):
        torch.func.vmap(lambda n: flash_hog.paged_cache_extend(new_tokens=1, **{**x, "lengths": n}))(torch.ones(2, 3, dtype=torch.int32))


@pytest.mark.parametrize("kind", [BF16, E4M3], ids=["bf16", "e4m3"])
@pytest.mark.parametrize("device", ["cuda", "cpu"])
def test_fake_tensors(device, kind):
    with FakeTensorMode():
        x = cpu(kind, device)
        free = flash_hog.paged_cache_extend(new_tokens=x["lengths"] * 1, **x)
        assert free.shape == () and free.dtype == torch.int32
        means = torch.zeros(4, 2, 64, device=device)
        got = flash_hog.paged_cache_compact(**x, num_pages=9, key_means=means)
        assert got[0].shape == (9, 2, 16, 64) and got[0].dtype == kind and got[4].shape == (9, 2, 64)
        assert (got[2] is None) == (kind == BF16) and got[5].shape == (3, 2)


@pytest.mark.parametrize("seed", range(40))
def test_oracle_keeps_rows_apart(seed):
    """After a step no page that a row writes next is anyone else's, and what every row held is still there."""
    page, pages, width = 16, 60, 5
    table, lengths, parents, new = ref.scenario(seed, 9, width, pages, page, wild=False)
    after, grown, left, copies = ref.extend(table, lengths, parents, new, pages, page)
    slots = {(p, r): (p, r) for p in range(pages) for r in range(page)}
    for source, target, rows in copies:
        slots.update({(target, r): slots[source, r] for r in range(rows)})
    written = set()
    for b, row in enumerate(after):
        parent = b if parents is None else parents[b]
        held = lengths[parent]
        for s in range(min(held, width * page)):
            assert slots[row[s // page], s % page] == (table[parent][s // page], s % page)
        for s in range(held, min(grown[b], width * page)):
            at = row[s // page], s % page
            if at[0] >= 0:
                assert at not in written
                written.add(at)
    for b, row in enumerate(after):
        parent = b if parents is None else parents[b]
        assert not written & {(row[s // page], s % page) for s in range(min(lengths[parent], width * page))}
    assert left <= pages
