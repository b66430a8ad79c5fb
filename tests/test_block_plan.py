"""csrc/fhog_block_plan.h, built with the host compiler: what attention of many tokens over chosen blocks indexes stays
inside the arrays that its plan lays out, wherever a sequence's tokens lie among the slabs."""

from __future__ import annotations

import ctypes
import random
import shutil
import subprocess

import pytest

from rules_host import CSRC

SOURCE = r"""
#include "fhog_block_plan.h"
namespace {
constexpr int kWays = 8;  // of block_items_kernel
int cut(int x, int total) { return x < 0 ? 0 : x > total ? total : x; }
}
extern "C" {
void plan(int batch, int total, int heads, int kv_heads, int head_dim, int width, int blocks, long* out) {
  const fhog::BlockChunkPlan p = fhog::block_chunk_plan(batch, total, heads, kv_heads, head_dim, width, blocks);
  out[0] = p.slab, out[1] = p.lists, out[2] = p.masks, out[3] = p.groups, out[4] = p.entries, out[5] = p.items;
  out[6] = p.parts, out[7] = (long)p.bytes;
}
int rule(int batch, int total, int heads, int kv_heads, int head_dim, int page, int width, int blocks) {
  return fhog::block_chunk_rule(batch, total, heads, kv_heads, head_dim, page, width, blocks, false);
}
// All slabs and sequences: the largest and smallest group that a list visits, less the slab's groups and 0 (out[0] < 0,
// out[1] >= 0), the largest index into masks and before, and how many packed tokens were in no way's groups, or in two.
void walk(const int* offsets, int batch, int total, int slab, int kv_heads, int width, long* out) {
  out[0] = -1, out[1] = 0, out[2] = -1, out[3] = 0;
  long seen = 0;
  for (int token0 = 0; token0 < total; token0 += slab) {
    const int tokens = total - token0 < slab ? total - token0 : slab, groups = (tokens + 63) / 64;
    for (int b = 0; b < batch; ++b) {
      const fhog::IndexRange of = fhog::slab_range(cut(offsets[b], total), cut(offsets[b + 1], total), token0, tokens);
      if (of.begin < 0 || of.end > tokens || of.begin > of.end) out[3] += 1l << 40;
      for (int way = 0; way < kWays; ++way) {
        const fhog::IndexRange g = fhog::list_groups(of, way, kWays);
        if (g.begin >= g.end) continue;
        if (g.end - 1 - groups > out[0]) out[0] = g.end - 1 - groups;
        if (g.begin < out[1]) out[1] = g.begin;
        const long at = ((long)(kv_heads - 1) * groups + g.end - 1) * width + width - 1;
        if (at > out[2]) out[2] = at;
        const int lo = 64 * g.begin > of.begin ? 64 * g.begin : of.begin, hi = 64 * g.end < of.end ? 64 * g.end : of.end;
        seen += hi - lo;
      }
    }
  }
  for (int b = 0; b < batch; ++b) {
    const int n = cut(offsets[b + 1], total) - cut(offsets[b], total);
    if (n > 0) seen -= n;
  }
  out[3] += seen < 0 ? -seen : seen;
}
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++") or shutil.which("clang++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    where = tmp_path_factory.mktemp("plan")
    (where / "plan.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-std=c++20", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", f"-I{CSRC}",
                    str(where / "plan.cpp"), "-o", str(where / "plan.so")], check=True)
    return ctypes.CDLL(str(where / "plan.so"))


def plan(lib, *args):
    out = (ctypes.c_long * 8)()
    lib.plan(*args, out)
    return dict(zip(("slab", "lists", "masks", "groups", "entries", "items", "parts", "bytes"), out))


def check_walk(lib, offsets, total, slab, kv_heads, width, masks):
    out = (ctypes.c_long * 4)()
    lib.walk((ctypes.c_int * len(offsets))(*offsets), len(offsets) - 1, total, slab, kv_heads, width, out)
    over, least, most, wrong = out
    assert over < 0 and least >= 0 and most < masks and wrong == 0, (offsets, total, slab)


# (heads, kv_heads, head_dim, width, blocks), and lengths: sequences that start behind the first slab, off a multiple of 64
@pytest.mark.parametrize("shape,new", [((32, 8, 128, 128, 16), [4001] * 4), ((8, 1, 128, 1024, 32), [9001, 9003, 9007, 8999]),
                                       ((32, 8, 128, 1024, 16), [31000, 1000, 5, 5]), ((32, 8, 128, 1024, 16), [99000, 1000, 5, 5]),
                                       ((8, 4, 64, 256, 64), [5001, 1, 0, 4900, 64, 3])], ids=str)
def test_sequences_behind_a_slab(rules, shape, new):
    heads, kv_heads, head_dim, width, blocks = shape
    offsets = [0]
    for n in new:
        offsets.append(offsets[-1] + n)
    assert rules.rule(len(new), offsets[-1], heads, kv_heads, head_dim, 64, width, blocks)
    p = plan(rules, len(new), offsets[-1], heads, kv_heads, head_dim, width, blocks)
    assert 0 < p["slab"] < offsets[-1] and p["slab"] % 64 == 0
    check_walk(rules, offsets, offsets[-1], p["slab"], kv_heads, width, p["masks"])


def test_any_offsets(rules):
    """Rising, falling and outside the packed rows; slabs from 64 tokens to all of them."""
    rng = random.Random(7)
    for _ in range(4000):
        total, batch = rng.choice([1, 63, 64, 65, 700, 5000, 40000]), rng.randint(1, 6)
        slab = min(total, 64 * rng.choice([1, 2, 7, 63, 125, 700]))
        kv_heads, width = rng.choice([1, 2, 8]), rng.choice([1, 3, 500])
        masks = kv_heads * -(-slab // 64) * width
        offsets = [rng.choice([rng.randint(0, total), rng.randint(-5, total + 5), -2 ** 31, 2 ** 31 - 1]) for _ in range(batch + 1)]
        if rng.random() < 0.7:
            offsets.sort()
        check_walk(rules, offsets, total, slab, kv_heads, width, masks)


# (batch, total, heads, kv_heads, head_dim, page, width, blocks): small outputs beside wide masks
WIDE = [(1, 131072, 8, 8, 64, 128, 4096, 4), (1, 262144, 4, 4, 64, 32, 8192, 8), (1, 1 << 20, 1, 1, 64, 128, 8192, 4)]


def test_workspace_bound(rules):
    """At most 1.1 GiB: the outputs and masks of a slab within 1 GiB; entries and items, of at most 1056 bytes for
    a tile of at least 65 rows of 264 bytes of outputs, and of 1060 for each of 32768 lists, are 9.5 % more."""
    rng, taken = random.Random(3), 0
    cases = list(WIDE)
    for _ in range(60000):
        kv_heads, group = rng.choice([1, 2, 4, 8, 12, 32]), rng.choice([1, 2, 3, 4, 8, 16, 43, 64, 65, 128])
        cases.append((rng.choice([1, 2, 16, 100]), int(2 ** rng.uniform(4, 21)), group * kv_heads, kv_heads, rng.choice([64, 128, 256]),
                      1 << rng.randint(4, 10), int(2 ** rng.uniform(0, 13)), int(2 ** rng.uniform(0, 8))))
    for batch, total, heads, kv_heads, head_dim, page, width, blocks in cases:
        if not rules.rule(batch, total, heads, kv_heads, head_dim, page, width, blocks):
            continue
        taken += 1
        p = plan(rules, batch, total, heads, kv_heads, head_dim, width, blocks)
        assert p["bytes"] <= 1.1 * 2 ** 30, (batch, total, heads, kv_heads, head_dim, page, width, blocks)
        assert p["slab"] == total or (p["slab"] >= 64 and p["slab"] % 64 == 0)
    assert taken > 5000
    assert all(rules.rule(*c[:6], *c[6:]) for c in WIDE)
