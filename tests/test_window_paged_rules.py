"""The rules of csrc/fhog_grid.h that split windowed and paged attention, built with the host
compiler: every pair of a sink and a query falls into one chunk, every packed row into one
tile, and no tile of rows reads more than its splits cover."""

from __future__ import annotations

import ctypes
import random
import shutil
import subprocess

import pytest

from rules_host import CSRC, CUS

SOURCE = r"""
#include "fhog_grid.h"
extern "C" {
void chunks(int nq, int nk, int coff, int window, int sinks, int row_bytes, int heads, int pairs, int* out) {
  const fhog::SinkChunks c = fhog::sink_chunks(fhog::Mask{true, nq, nk, coff}, window, sinks, row_bytes, heads, pairs);
  out[0] = c.apart, out[1] = c.step, out[2] = c.count;
}
void plan(int batch, int total, int single, int heads, int kv_heads, int d, long capacity, int window, int sinks, int cus,
          long* out) {
  const fhog::PagedPlan p = fhog::paged_plan(batch, total, single, heads, kv_heads, d, capacity, window, sinks, cus);
  out[0] = p.rows, out[1] = p.slots, out[2] = p.splits, out[3] = p.split_tiles, out[4] = p.parts, out[5] = p.longest_first;
}
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++") or shutil.which("clang++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    where = tmp_path_factory.mktemp("rules")
    (where / "rules.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-std=c++20", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}",
                    str(where / "rules.cpp"), "-o", str(where / "rules.so")], check=True)
    lib = ctypes.CDLL(str(where / "rules.so"))
    lib.plan.argtypes = [ctypes.c_int] * 6 + [ctypes.c_long] + [ctypes.c_int] * 3 + [ctypes.POINTER(ctypes.c_long)]
    return lib


def sink_chunks(lib, *args):
    out = (ctypes.c_int * 3)()
    lib.chunks(*args, out)
    return bool(out[0]), out[1], out[2]


def plan(lib, *args):
    out = (ctypes.c_long * 6)()
    lib.plan(*args, out)
    return dict(zip(("rows", "slots", "splits", "split_tiles", "parts", "longest_first"), out))


def test_sink_chunks_cover_the_queries(rules):
    rng = random.Random(4)
    for _ in range(3000):
        nq, nk = rng.choice([1, 40, 700, 5000, 1 << 20]), rng.choice([1, 40, 700, 5000, 1 << 20])
        coff = rng.choice([0, nk - nq])
        window, sinks = rng.randint(1, max(nq, nk)), rng.randint(0, nk)
        pairs = rng.choice([1, 8, 64])
        apart, step, count = sink_chunks(rules, nq, nk, coff, window, sinks, rng.choice([128, 256, 512]), pairs, pairs)
        first = window - coff  # the first query whose window lies behind key 0
        if sinks == 0 or first >= nq:
            assert count == 0
            continue
        begin = max(0, first) // 32 * 32
        assert step > 0 and step % 32 == 0 and count >= 1
        assert begin + count * step >= nq > begin + (count - 1) * step
        assert count * sinks <= (nq + 1) // 2 + sinks  # the parts' rows


def test_largest_sizes(rules):
    most = 1 << 30
    assert sink_chunks(rules, most, most, 0, 1, most, 128, 1, 1)[1:] == (most, 1)
    p = plan(rules, 1, 1 << 23, 0, 128, 1, 256, most, 0, 0, CUS)
    assert p["slots"] > 0 and p["splits"] >= 1
    p = plan(rules, (1 << 24) - 1, (1 << 24) - 1, 1, 16, 1, 64, most, most, most, CUS)
    assert p["slots"] == (1 << 24) - 1 and p["splits"] == 1


def span_tiles(first_pos, last_pos, length, window, sinks):
    """32-key tiles that the rows at these positions read (PageSpan)."""
    hi = max(0, min(length, last_pos + 1))
    lo = min(max(0, first_pos - window + 1), hi) if window else 0
    behind = max(0, min(sinks, lo)) if window else 0
    return (behind + 31) // 32 + (hi - lo // 16 * 16 + 31) // 32 if hi else 0


@pytest.mark.parametrize("cus", [CUS, 0, 64])
def test_tiles_cover_rows_and_splits_cover_keys(rules, cus):
    rng = random.Random(7)
    for _ in range(1500):
        kv = rng.choice([1, 2, 8])
        group = rng.choice([1, 2, 3, 4, 7, 8, 16, 17, 40, 150])
        batch = rng.choice([1, 2, 5, 40])
        single = rng.random() < 0.4
        pages = rng.choice([1, 3, 20, 300, 2048])
        capacity = 16 * pages
        counts = [1] * batch if single else [rng.choice([0, 1, 2, 15, 16, 17, 100, 400]) for _ in range(batch)]
        total = sum(counts)
        if total == 0:
            continue
        window = rng.choice([0, 0, 1, 30, 500])
        sinks = rng.choice([0, 1, 40, 400]) if window else 0
        p = plan(rules, batch, total, single, group * kv, kv, rng.choice([64, 128, 256]), capacity, window, sinks, cus)
        rows = p["rows"]
        assert p["splits"] >= 1 and p["splits"] * rows <= 2048 and p["split_tiles"] >= 1
        if p["longest_first"]:  # one lane a sequence, no splits, nothing that cuts keys off
            assert rows > 16 and 1 < batch <= 64 and p["splits"] == 1 and window == 0
        assert p["parts"] == (p["slots"] * kv * p["splits"] * rows if p["splits"] > 1 else 0)
        begin, seen = 0, 0
        for b, count in enumerate(counts):
            first = b * -(-group // rows) if single else begin * group // rows + b
            after = first + -(-group // rows) if single else (begin + count) * group // rows + b + 1
            assert first >= seen and after <= p["slots"]  # no two sequences share a tile
            tiles = -(-count * group // rows)
            assert first + tiles <= after
            seen = first + tiles
            length = rng.choice([capacity, max(count, 1), min(capacity, max(count, capacity // 2 + 5))])
            for tile in {0, tiles - 1} if tiles else ():
                last = min(count * group, (tile + 1) * rows) - 1
                positions = [length - count + r // group for r in (tile * rows, last)]
                assert span_tiles(*positions, min(length, capacity), window, sinks) <= p["splits"] * p["split_tiles"]
            begin += count


def test_variants(rules):
    """Rows of a tile and splits at the sizes that the rules' comments name."""
    def rows(batch, new, heads, kv, d, keys, window=0):
        p = plan(rules, batch, batch * new, new == 1, heads, kv, d, keys, window, 0, CUS)
        return p["rows"], p["splits"]

    assert rows(16, 1, 32, 8, 128, 32768) == (16, 16)
    assert rows(1, 1, 16, 4, 64, 32768)[0] == 16
    assert rows(64, 1, 32, 8, 128, 4096)[1] == 1
    assert rows(8, 512, 32, 8, 128, 8192, 2048) == (128, 1)
    assert rows(32, 64, 16, 4, 64, 4096)[0] == 64
    assert rows(1, 64, 32, 8, 128, 32768) == (64, 13)
