"""Norms with rotation, the paged cache's allocator and attention over chosen blocks: performance
cases of their operators.

listed() names the cases, draw(rng) gives one more of the same ranges, prepare(case, seed)
makes the inputs on the GPU, run(state) is one pass, work(case) its least bytes and flops,
exact(case, seed) the outputs in 64 bits.

The operators (`op`):

  rotary   qk_norm_rotary: the rows of queries and keys, each head's own, divided by their root
           mean square, times a weight, and rotated in pairs by their position's angles. `kind`
           forward: no autograd; train: with the gradients for an upstream gradient; hvp: the
           gradients and their derivative along tangents of what they belong to.
  blocks   a serving step over chosen blocks: paged_key_means (the mean key of each page that the new
           tokens fill), paged_block_select (for each new token and key/value head the pages whose
           mean has the largest product with the sum of its queries, the first and the last ones
           besides), paged_block_attention (attention over these pages).
  extend   paged_cache_extend: rows of a page table become those of their parents and grow by new
           tokens; a shared last page is copied first, and pages that no row uses are handed out.
           Before it, lengths go back to what they were, as after drafted tokens that were rejected.
  compact  paged_cache_compact: the used pages of a cache, in their order, as the first of a new one.

A cache is (pages, kv_heads, page_size, head_dim); an e4m3 cache has an e8m0 scale (a power of
two) for each key and value row, (pages, kv_heads, page_size).
"""

import math
import os
import sys

import numpy as np
import torch

own = False

_PACKAGE_ROOT = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-hog_amd")

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
_EPS = 1e-6


def _rotary(name, kind, batch, n, heads, kv_heads, head_dim, rotated, dtype, where, interleaved=False, norm=True,
            fused=False):
    """`rotated` of head_dim columns turn. `where` positions come from: start (0 on), given (a tensor) or
    cache (the lengths of `batch` sequences with n new tokens each, packed). fused: queries and keys lie
    in one tensor with the values."""
    case = {"op": "rotary", "kind": kind, "batch": batch, "n": n, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "rotated": rotated, "dtype": dtype, "where": where, "interleaved": interleaved,
            "norm": norm, "fused": fused}
    return {"name": name, **case} if name else case


def _blocks(name, batch, new_min, new, length_min, length, heads, kv_heads, head_dim, dtype, cache, page, chosen,
            first=1, last=1):
    """`new` tokens at most (new_min at least) in each of `batch` sequences that hold length_min to
    `length` tokens with the new ones; each attends to `chosen` pages."""
    case = {"op": "blocks", "batch": batch, "new_min": new_min, "new": new, "length_min": length_min,
            "length": length, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype,
            "cache": cache, "page": page, "chosen": chosen, "first": first, "last": last}
    return {"name": name, **case} if name else case


def _extend(name, batch, parents, length_min, length, new, kv_heads, head_dim, cache, page):
    """`parents` of `batch` sequences, of length_min to `length` tokens, go on in all rows, by `new`
    tokens each."""
    case = {"op": "extend", "batch": batch, "parents": parents, "length_min": length_min, "length": length, "new": new,
            "kv_heads": kv_heads, "head_dim": head_dim, "cache": cache, "page": page}
    return {"name": name, **case} if name else case


def _compact(name, batch, ended, length_min, length, kv_heads, head_dim, cache, page):
    """`batch` sequences of length_min to `length` tokens, of which `ended` have ended since."""
    case = {"op": "compact", "batch": batch, "ended": ended, "length_min": length_min, "length": length,
            "kv_heads": kv_heads, "head_dim": head_dim, "cache": cache, "page": page}
    return {"name": name, **case} if name else case


def listed():
    return [
        # The next token of one conversation: latency.
        _rotary("rotary_token_b1_h16_kv4_d64", "forward", 1, 1, 16, 4, 64, 64, "bf16", "cache"),
        # A training step in full precision, no size a multiple of a tile, half of each row rotated.
        _rotary("rotary_train_b1_n1333_h8_d64_fp32", "train", 1, 1333, 8, 8, 64, 32, "fp32", "start"),
        # A training step with grouped heads on the views of a joint projection, documents packed into rows,
        # neighbouring columns rotated.
        _rotary("rotary_train_b2_n4001_h32_kv8_d128_fp16", "train", 2, 4001, 32, 8, 128, 128, "fp16", "given",
                interleaved=True, fused=True),
        # A curvature probe on one long sequence.
        _rotary("rotary_hvp_b1_n16384_h12_d64", "hvp", 1, 16384, 12, 12, 64, 64, "bf16", "start"),
        # The next token of one conversation over a few of its pages: latency.
        _blocks("blocks_token_b1_len8000_h16_kv4_d64", 1, 1, 1, 8000, 8000, 16, 4, 64, "bf16", "bf16", 16, 32),
        # The next token of a batch of very long, unequal conversations over a quantised cache.
        _blocks("blocks_token_b16_len65536_h32_kv8_d128_e4m3", 16, 1, 1, 4000, 65536, 32, 8, 128, "bf16", "e4m3", 64,
                64, 1, 2),
        # Short and longer pieces of prompts together, on contexts of unequal length.
        _blocks("blocks_chunk_b4_new1000_len8192_h32_kv8_d128", 4, 17, 1000, 1500, 8192, 32, 8, 128, "bf16", "bf16",
                64, 16, 1, 2),
        # A long prompt's last quarter over a quantised cache, without grouping.
        _blocks("blocks_chunk_b1_new4096_len16384_h12_d64_fp16_e4m3", 1, 4096, 4096, 16384, 16384, 12, 12, 64, "fp16",
                "e4m3", 64, 16),
        # One conversation goes on by a token.
        _extend("extend_b1_len1000_kv4_d64", 1, 1, 1000, 1000, 1, 4, 64, "bf16", 16),
        # A beam search's step: each of 16 prompts goes on in eight rows.
        _extend("extend_b128_of16_len4096_kv8_d128", 128, 16, 500, 4096, 1, 8, 128, "bf16", 128),
        # A small server's cache after some conversations have ended.
        _compact("compact_b8_len500_kv4_d64", 8, 3, 100, 500, 4, 64, "bf16", 16),
        # A large one's, quantised.
        _compact("compact_b32_len16384_kv8_d128_e4m3", 32, 12, 2000, 16384, 8, 128, "e4m3", 64),
    ]


# ------------------------------------------------------------------ more cases

def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_rotary(rng):
    kind = rng.choice(("forward", "train", "hvp"))
    where = rng.choice(("start", "given", "cache")) if kind == "forward" else rng.choice(("start", "given"))
    kv_heads = rng.choice((1, 2, 4, 8, 12, 16))
    head_dim = rng.choice((64, 64, 80, 128, 128, 256))
    rotated = rng.choice((head_dim, head_dim, head_dim // 2, head_dim // 4))
    return _rotary(None, kind, _log_int(rng, 1, 32), _log_int(rng, 1, 16384), kv_heads * rng.choice((1, 1, 2, 4)),
                   kv_heads, head_dim, rotated, rng.choices(("bf16", "fp16", "fp32"), (5, 3, 2))[0], where,
                   rng.random() < 0.3, rng.random() < 0.8, rng.random() < 0.5)


def _draw_blocks(rng):
    batch = _log_int(rng, 1, 32)
    length = _log_int(rng, 64, 65536)
    length_min = max(1, int(length * rng.uniform(0.1, 1.0)))
    new = 1 if rng.random() < 0.5 else min(length_min, _log_int(rng, 2, 4096))
    new_min = max(1, int(new * rng.uniform(0.1, 1.0)))
    kv_heads = rng.choice((1, 2, 4, 8, 12))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    first, last = rng.choice((0, 1, 1, 2)), rng.choice((1, 1, 2))
    return _blocks(None, batch, new_min, new, length_min, length, kv_heads * rng.choice((1, 2, 4, 8)), kv_heads,
                   rng.choice((64, 128, 128, 256)), dtype, rng.choice((dtype, "e4m3")), rng.choice((16, 32, 64, 128)),
                   rng.choice((4, 8, 15, 16, 32, 64)), first, last)


def _draw_extend(rng):
    batch = _log_int(rng, 1, 256)
    length = _log_int(rng, 16, 16384)
    return _extend(None, batch, max(1, batch // rng.choice((1, 1, 2, 4, 8))), max(1, int(length * rng.uniform(0.1, 1.0))),
                   length, rng.choice((0, 1, 1, 5, 300)), rng.choice((1, 2, 4, 8, 16)), rng.choice((64, 128, 256)),
                   rng.choice(("bf16", "fp16", "e4m3")), rng.choice((16, 32, 64, 128, 256)))


def _draw_compact(rng):
    batch = _log_int(rng, 1, 64)
    length = _log_int(rng, 16, 16384)
    return _compact(None, batch, int(batch * rng.uniform(0, 0.9)), max(1, int(length * rng.uniform(0.1, 1.0))), length,
                    rng.choice((1, 2, 4, 8, 16)), rng.choice((64, 128, 256)), rng.choice(("bf16", "fp16", "e4m3")),
                    rng.choice((16, 32, 64, 128, 256)))


def draw(rng):
    """One case of the ranges above: 1 to 16384 tokens' rows, 64 to 65536 cached tokens, 1 to 256 sequences
    (sizes over their logarithm, odd ones among them), 1 to 64 heads, grouped or not, each dtype,
    head dim, page size and kind."""
    biggest = {}
    for case in listed():
        best = biggest.setdefault(case["op"], {})
        for key, value in _costs(case).items():
            best[key] = max(best.get(key, 0), value)
    while True:
        case = rng.choices((_draw_rotary, _draw_blocks, _draw_extend, _draw_compact), (3, 4, 2, 1))[0](rng)
        costs = _costs(case)
        if all(v <= biggest[case["op"]][key] for key, v in costs.items()) and case.get("heads", 0) <= 64:
            return case


def _costs(case):
    """What a drawn case may not have more of than the listed ones."""
    costs = work(case)
    if case["op"] == "blocks":  # the plain form's keys, and the cache
        new, lengths = _counts(case)
        keys = case["chosen"] * case["page"]
        costs["keys"] = int(new.sum()) * case["kv_heads"] * keys * case["head_dim"]
        costs["scores"] = case["batch"] * case["new"] * case["kv_heads"] * _pages_per_sequence(case)
        costs["cache"] = int(lengths.sum()) * case["kv_heads"] * case["head_dim"]
    elif case["op"] != "rotary":
        costs["cache"] = _pool(case) * case["kv_heads"] * case["page"] * case["head_dim"] * _BYTES[case["cache"]]
    return costs


# ------------------------------------------------------------------ sizes that a case implies

def _spread(lo, hi, count):
    """`count` whole numbers from hi down to lo."""
    return np.array([hi if count == 1 else hi - (hi - lo) * i // (count - 1) for i in range(count)])


def _counts(case):
    """New tokens and lengths of the sequences, before a seed puts them in an order."""
    return _spread(case["new_min"], case["new"], case["batch"]), _spread(case["length_min"], case["length"], case["batch"])


def _pages_per_sequence(case):
    return -(-case["length"] // case["page"]) + 1


def _tokens(case):
    """Tokens of a rotary case, as their tensors' leading sizes."""
    return (case["batch"] * case["n"],) if case["where"] == "cache" else (case["batch"], case["n"])


def _children(case):
    """The parent of each row of an extend case: row i goes on from row i % parents."""
    return np.arange(case["batch"]) % case["parents"]


def _extend_lengths(case):
    """The rows' lengths before the call; only those of the parents count."""
    lengths = _spread(case["length_min"], case["length"], case["parents"])
    return lengths[_children(case)]


def _extend_width(case):
    return -(-(case["length"] + case["new"]) // case["page"]) + 2


def _pool(case):
    """Pages of the cache."""
    if case["op"] == "extend":
        lengths = _extend_lengths(case)
        parents = lengths[:case["parents"]]
        held = int((-(-parents // case["page"])).sum())
        each = -(-(case["length"] + case["new"]) // case["page"]) - case["length"] // case["page"] + 1
        return held + case["batch"] * each + 5
    lengths = _spread(case["length_min"], case["length"], case["batch"])
    return int((-(-lengths // case["page"])).sum()) + 3


def work(case):
    if case["op"] == "rotary":
        tokens = case["batch"] * case["n"]
        rows = tokens * (case["heads"] + case["kv_heads"])
        # x -> y; x, dy -> y, dx; x, dy, tangents -> dx, and the derivatives for x and dy
        tensors, flops = {"forward": (2, 8), "train": (4, 24), "hvp": (6, 60)}[case["kind"]]
        return {"bytes": tensors * rows * case["head_dim"] * _BYTES[case["dtype"]], "flops": flops * rows * case["head_dim"]}
    d, kv = case["head_dim"], case["kv_heads"]
    row = 2 * (d * _BYTES[case["cache"]] + (1 if case["cache"] == "e4m3" else 0))  # a token's key and value of a head
    page = case["page"]
    if case["op"] == "blocks":
        new, lengths = _counts(case)
        item = _BYTES[case["dtype"]]
        scored = pairs = full = keys = 0
        for count, length in zip(new, lengths):
            p = np.arange(length - count, length, dtype=np.int64)
            seen = np.minimum(p // page + 1, case["chosen"])
            scored += int(np.maximum(p // page + 1 - case["first"] - case["last"], 0).sum())
            pairs += int(((seen - 1) * page + p % page + 1).sum())
            full += int(length // page)
            keys += min(int(length), int(((seen - 1) * page + p % page + 1).sum()))
        total = int(new.sum())
        chosen = 4 * total * kv * case["chosen"]
        bytes_ = (4 * full * kv * d + keys * kv * row + 2 * total * case["heads"] * d * item + chosen
                  + 4 * case["batch"] * _pages_per_sequence(case))
        return {"bytes": bytes_, "flops": 4 * d * pairs * case["heads"] + 2 * d * scored * kv}
    if case["op"] == "extend":
        lengths = _extend_lengths(case)
        parents = _children(case)
        shared = [i for i in range(case["batch"]) if i >= case["parents"] and case["new"] and lengths[i] % page]
        held = int(sum(lengths[i] % page for i in shared if parents[i] != i))
        table = int((-(-(lengths + case["new"]) // page)).sum())
        return {"bytes": 2 * held * kv * row + 8 * table + 12 * case["batch"], "flops": 2 * table}
    lengths = _spread(case["length_min"], case["length"], case["batch"])[case["ended"]:]
    used = int((-(-lengths // page)).sum())
    pages = used * kv * page * row
    return {"bytes": 2 * pages + 8 * used, "flops": 2 * used}


# ------------------------------------------------------------------ inputs

def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _exponent(amax):
    """The e8m0 code of each row's scale from its largest magnitude (fp32): 2^(code - 127)."""
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa 2^exponent, mantissa in [1/2, 1)
    code = exponent - 1 - 8 + (mantissa > 0.875).to(exponent.dtype) + 127
    return torch.where(amax > 0, code, torch.ones_like(code)).clamp(1, 254).to(torch.uint8)


def _scales(code):
    """The powers of two that e8m0 codes (bytes, 1 to 254) stand for, in fp32."""
    return (code.to(torch.int32) << 23).view(torch.float32)


def _quantise(x):
    """e4m3 values and e8m0 scales of the rows of x (their last axis), as bytes."""
    code = _exponent(x.abs().amax(-1))
    return (x / _scales(code)[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), code


def _fill(state, gen, pages, case, dtype):
    """Keys and values of `pages` pages, of rows of unlike magnitude."""
    kv, page, d = case["kv_heads"], case["page"], case["head_dim"]
    for n in ("k", "v"):
        rows = torch.randn((pages, kv, page, d), generator=gen, device="cuda")
        rows *= torch.exp(0.5 * torch.randn((pages, kv, page, 1), generator=gen, device="cuda")) * 0.7
        if n == "k" and case["op"] == "blocks":  # a page's keys have something in common
            rows += 0.4 * torch.randn((pages, kv, 1, d), generator=gen, device="cuda")
        if case["cache"] == "e4m3":
            values, code = _quantise(rows)
            state[n + "_cache"] = values.view(torch.float8_e4m3fn)
            state[n + "_scale"] = code.view(torch.float8_e8m0fnu)
        else:
            state[n + "_cache"], state[n + "_scale"] = rows.to(dtype), None
        del rows


def _paged_table(order, lengths, page, width, pages):
    """Pages of the sequences in random order, -1 where there is none."""
    used = -(-lengths // page)
    table = np.full((len(lengths), width), -1, dtype=np.int32)
    ids, first = order.permutation(pages), 0
    for b, n in enumerate(used):
        table[b, :n] = ids[first:first + n]
        first += n
    return table, ids[first:]


def _device(x):
    return torch.from_numpy(np.ascontiguousarray(x).astype(np.int32)).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    order = np.random.RandomState(seed)
    return {"rotary": _prepare_rotary, "blocks": _prepare_blocks, "extend": _prepare_extend,
            "compact": _prepare_compact}[case["op"]](case, gen, order)


def _prepare_rotary(case, gen, order):
    dtype, d, h, kv = _DTYPES[case["dtype"]], case["head_dim"], case["heads"], case["kv_heads"]
    tokens = _tokens(case)
    state = {"case": case}
    rows = torch.randn((*tokens, h + 2 * kv, d), generator=gen, device="cuda")
    rows = (rows * torch.exp(0.5 * torch.randn((*tokens, h + 2 * kv, 1), generator=gen, device="cuda"))).to(dtype)
    parts = rows[..., :h, :], rows[..., h:h + kv, :]
    state["q"], state["k"] = parts if case["fused"] else (x.contiguous() for x in parts)
    for n in ("wq", "wk"):
        state[n] = (1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(dtype) if case["norm"] else None
    state["frequencies"] = (10000.0 ** (-torch.arange(0, case["rotated"], 2, dtype=torch.float64) / case["rotated"])).float().cuda()
    state["positions"] = state["lengths"] = state["offsets"] = None
    if case["where"] == "given":  # documents of unequal length, one behind the other
        positions = np.zeros(tokens, dtype=np.int32)
        for b in range(tokens[0]):
            at = 0
            while at < tokens[1]:
                n = min(tokens[1] - at, 1 + order.randint(tokens[1]))
                positions[b, at:at + n] = np.arange(n) + order.randint(2) * order.randint(100000)
                at += n
        state["positions"] = _device(positions)
    elif case["where"] == "cache":
        state["lengths"] = _device(case["n"] + order.randint(100000, size=case["batch"]))
        if case["n"] > 1:
            state["offsets"] = _device(np.arange(case["batch"] + 1) * case["n"])
    if case["kind"] != "forward":
        for n, like in (("cq", "q"), ("ck", "k")):
            state[n] = _normal(gen, state[like].shape, dtype)
        for n in ("q", "k", "wq", "wk"):
            if state[n] is not None:
                state[n] = state[n].detach().requires_grad_()
        if case["kind"] == "hvp":
            for n in ("cq", "ck"):
                state[n].requires_grad_()
            for n in ("q", "k", "wq", "wk"):
                state["t" + n] = None if state[n] is None else _normal(gen, state[n].shape, dtype)
    return state


def _prepare_blocks(case, gen, order):
    dtype, page, kv, d = _DTYPES[case["dtype"]], case["page"], case["kv_heads"], case["head_dim"]
    new, lengths = _counts(case)
    at = order.permutation(case["batch"])  # which sequence is how long has nothing to do with its place
    new, lengths = new[at], lengths[at]
    pages = int((-(-lengths // page)).sum()) + 3
    table, _ = _paged_table(order, lengths, page, _pages_per_sequence(case), pages)
    state = {"case": case, "table": _device(table), "lengths": _device(lengths), "offsets": None}
    if case["new"] > 1:
        state["offsets"] = _device(np.concatenate([[0], np.cumsum(new)]))
    _fill(state, gen, pages, case, dtype)
    total = int(new.sum())
    state["q"] = _normal(gen, (total, case["heads"], d), dtype)
    means = torch.zeros((pages, kv, d), device="cuda")
    for b in range(case["batch"]):  # the pages that were full before
        ids = torch.from_numpy(table[b, :(lengths[b] - new[b]) // page]).cuda().long()
        for part in ids.split(256):
            means[part] = (_page_rows(state, "k", part).double().sum(2) / page).float()
        if lengths[b] % page:  # slots that hold no token yet may hold anything
            last = int(table[b, lengths[b] // page])
            for n in ("k", "v"):
                if case["cache"] == "e4m3":
                    state[n + "_cache"].view(torch.uint8)[last, :, lengths[b] % page:] = 0x7F
                else:
                    state[n + "_cache"][last, :, lengths[b] % page:] = float("nan")
    state["means"] = means
    return state


def _prepare_extend(case, gen, order):
    page = case["page"]
    state = {"case": case}
    pages = _pool(case)
    lengths = _extend_lengths(case)
    _fill(state, gen, pages, case, _DTYPES.get(case["cache"]))
    held = np.where(np.arange(case["batch"]) < case["parents"], lengths, 0)
    table, _ = _paged_table(order, held, page, _extend_width(case), pages)
    state["table"], state["start"] = _device(table), _device(lengths)
    state["lengths"] = state["start"].clone()
    state["parents"] = None if case["parents"] == case["batch"] else _device(_children(case))
    return state


def _prepare_compact(case, gen, order):
    state = {"case": case}
    pages = _pool(case)
    lengths = _spread(case["length_min"], case["length"], case["batch"])
    table, _ = _paged_table(order, lengths, case["page"], _pages_per_sequence(case), pages)
    lengths[:case["ended"]] = 0
    at = order.permutation(case["batch"])
    _fill(state, gen, pages, case, _DTYPES.get(case["cache"]))
    state["table"], state["lengths"] = _device(table[at]), _device(lengths[at])
    state["num_pages"] = max(1, int((-(-lengths // case["page"])).sum()))
    return state


# ------------------------------------------------------------------ one pass

def run(s):
    op = s["case"]["op"]
    if op == "rotary":
        return _run_rotary(s)
    if op == "extend":
        s["lengths"].copy_(s["start"])
    if own:
        return {"blocks": _call_blocks, "extend": _call_extend, "compact": _call_compact}[op](s)
    return {"blocks": _plain_blocks, "extend": _plain_extend, "compact": _plain_compact}[op](s)


def _flash_hog():
    if _PACKAGE_ROOT not in sys.path:
        sys.path.insert(0, _PACKAGE_ROOT)
    import flash_hog

    return flash_hog


def _run_rotary(s):
    case = s["case"]
    apply = _call_rotary if own else _plain_rotary
    if case["kind"] == "forward":
        with torch.no_grad():
            return apply(s)
    leaves = [s[n] for n in ("q", "k", "wq", "wk") if s[n] is not None]
    out = apply(s)
    if case["kind"] == "train":
        return (*(y.detach() for y in out), *torch.autograd.grad(out, leaves, (s["cq"], s["ck"])))
    grads = torch.autograd.grad(out, leaves, (s["cq"], s["ck"]), create_graph=True)
    tangents = [s["t" + n] for n in ("q", "k", "wq", "wk") if s[n] is not None]
    # Without norms the gradients do not depend on the rows.
    wanted = (*leaves, s["cq"], s["ck"]) if case["norm"] else (s["cq"], s["ck"])
    products = torch.autograd.grad(grads, wanted, tangents)
    return (*(g.detach() for g in grads), *products)


def _call_rotary(s):
    case = s["case"]
    return _flash_hog().qk_norm_rotary(s["q"], s["k"], s["positions"], frequencies=s["frequencies"],
                                       query_weight=s["wq"], key_weight=s["wk"], eps=_EPS if case["norm"] else None,
                                       interleaved=case["interleaved"], lengths=s["lengths"],
                                       query_offsets=s["offsets"])


def _call_blocks(s):
    case, hog = s["case"], _flash_hog()
    hog.paged_key_means(s["k_cache"], s["means"], s["table"], s["lengths"], s["offsets"], key_scale=s["k_scale"])
    chosen = hog.paged_block_select(s["q"], s["means"], s["table"], s["lengths"], s["offsets"], page_size=case["page"],
                                    blocks=case["chosen"], first=case["first"], last=case["last"])
    out = hog.paged_block_attention(s["q"], chosen, s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["offsets"],
                                    key_scale=s["k_scale"], value_scale=s["v_scale"])
    return s["means"], chosen, out


def _call_extend(s):
    free = _flash_hog().paged_cache_extend(s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["case"]["new"],
                                           s["parents"], key_scale=s["k_scale"], value_scale=s["v_scale"])
    return (*_caches(s), s["table"], s["lengths"], free)


def _call_compact(s):
    got = _flash_hog().paged_cache_compact(s["k_cache"], s["v_cache"], s["table"], s["lengths"],
                                           num_pages=s["num_pages"], key_scale=s["k_scale"], value_scale=s["v_scale"])
    return tuple(x for x in got if x is not None)


def _caches(s):
    return tuple(s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale") if s[n] is not None)


# ------------------------------------------------------------------ plain forms

def _positions(s, tokens):
    """Positions of a rotary case's tokens, in 64 bits."""
    if s["positions"] is not None:
        return s["positions"].double()
    if s["lengths"] is None:
        return torch.arange(tokens[1], device="cuda", dtype=torch.float64)[None]
    n = tokens[0] // s["lengths"].shape[0]
    return (s["lengths"].double()[:, None] - n + torch.arange(n, device="cuda")).reshape(-1)


def _plain_rotary(s):
    case = s["case"]
    angle = _positions(s, _tokens(case))[..., None] * s["frequencies"].double()  # (..., rotated / 2)
    cos, sin = angle.cos().float()[..., None, :], angle.sin().float()[..., None, :]
    R, got = case["rotated"], []
    for n in ("q", "k"):
        x = s[n].float()
        if case["norm"]:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * s["w" + n].float()
        a, b = (x[..., 0:R:2], x[..., 1:R:2]) if case["interleaved"] else (x[..., :R // 2], x[..., R // 2:R])
        turned = a * cos - b * sin, b * cos + a * sin
        if case["interleaved"]:
            turned = (torch.stack(turned, -1).flatten(-2),)
        got.append(torch.cat([*turned, x[..., R:]], -1).to(s[n].dtype))
    return tuple(got)


def _page_rows(s, n, ids):
    """Rows of whole pages, dequantised, in fp32: (..., kv_heads, page, head_dim)."""
    x = s[n + "_cache"].view(torch.uint8)[ids].view(s[n + "_cache"].dtype).float()
    if s[n + "_scale"] is not None:
        x = x * _scales(s[n + "_scale"].view(torch.uint8)[ids])[..., None]
    return x


def _sequence_rows(s, total):
    """Of the packed rows: their sequences and their places among the sequence's new tokens; of the
    sequences: how many new tokens they have and where these start."""
    rows = torch.arange(total, device="cuda")
    offsets = s["offsets"]
    if offsets is None:
        offsets = torch.arange(total + 1, device="cuda")
    offsets = offsets.long()
    b = torch.searchsorted(offsets[1:].contiguous(), rows, right=True)
    return b, rows - offsets[b], offsets[1:] - offsets[:-1], offsets[:-1]


def _plain_means(s, counts):
    """The means of the pages that the new tokens fill, summed in 64 bits, so that their order is nothing."""
    page, means, lengths = s["case"]["page"], s["means"], s["lengths"].long()
    col = ((lengths - counts) // page)[:, None] + torch.arange(s["case"]["new"] // page + 1, device="cuda")
    filled = col < (lengths // page)[:, None]
    ids = s["table"].long().gather(1, torch.where(filled, col, torch.zeros_like(col)))
    mean = (_page_rows(s, "k", ids).double().sum(-2) / page).float()
    ids = torch.where(filled, ids, torch.full_like(ids, means.shape[0]))  # the others to a page that is dropped
    more = torch.cat([means, means[:1]])
    more[ids] = mean
    means.copy_(more[:-1])


def _plain_select(s, row_b, row_i, counts, starts):
    """Scores in 64 bits: which page is chosen hangs on them."""
    case, q = s["case"], s["q"]
    T, H, d = q.shape
    N, new, page = case["kv_heads"], case["new"], case["page"]
    lengths = s["lengths"].long()
    B, width = s["table"].shape
    i = torch.arange(new, device="cuda")
    qs = q.double().reshape(T, N, H // N, d).sum(2)
    qs = qs[(starts[:, None] + i).clamp(max=T - 1)].transpose(1, 2)  # (B, N, new, d)
    m = s["means"][s["table"].clamp(min=0).long()].double()  # (B, width, N, d)
    score = torch.matmul(qs, m.permute(0, 2, 3, 1).contiguous())  # (B, N, new, width)
    pos = (lengths - counts)[:, None] + i
    at = (pos // page)[:, None, :, None]  # the token's own page
    col = torch.arange(width, device="cuda")
    score = torch.where((col < case["first"]) | (col > at - case["last"]), torch.full_like(score, float("inf")), score)
    score = torch.where(col > at, torch.full_like(score, float("-inf")), score)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :case["chosen"]]
    best = torch.where(best > at, torch.full_like(best, width), best).sort(-1).values
    best = torch.where(best == width, torch.full_like(best, -1), best).to(torch.int32)
    if best.shape[-1] < case["chosen"]:
        best = torch.cat([best, best.new_full((*best.shape[:-1], case["chosen"] - best.shape[-1]), -1)], -1)
    return best.transpose(1, 2)[row_b, row_i].contiguous()


def _plain_blocks(s):
    case, q = s["case"], s["q"]
    T, H, d = q.shape
    N, page = case["kv_heads"], case["page"]
    row_b, row_i, counts, starts = _sequence_rows(s, T)
    _plain_means(s, counts)
    chosen = _plain_select(s, row_b, row_i, counts, starts)
    pos = s["lengths"].long()[row_b] - counts[row_b] + row_i
    out = torch.empty_like(q)
    head = torch.arange(N, device="cuda")[:, None]
    step = max(1, 2 ** 27 // (N * case["chosen"] * page * d))
    for t in range(0, T, step):
        block = chosen[t:t + step].long()  # (t, N, chosen)
        ids = s["table"].long()[row_b[t:t + step, None, None], block.clamp(min=0)].clamp(min=0)
        rows = []
        for n in ("k", "v"):
            x = s[n + "_cache"].view(torch.uint8)[ids, head].view(s[n + "_cache"].dtype).float()  # (t, N, chosen, page, d)
            if s[n + "_scale"] is not None:
                x = x * _scales(s[n + "_scale"].view(torch.uint8)[ids, head])[..., None]
            rows.append(x.flatten(2, 3))
        key = (block[..., None] * page + torch.arange(page, device="cuda")).flatten(2)
        mask = (block >= 0)[..., None].expand(*block.shape, page).flatten(2) & (key <= pos[t:t + step, None, None])
        k, v = rows
        v = torch.where(mask[..., None], v, torch.zeros_like(v))
        scores = torch.matmul(q[t:t + step].float().reshape(-1, N, H // N, d), k.transpose(-1, -2)) * d ** -0.5
        scores = torch.where(mask[:, :, None], scores, torch.full_like(scores, float("-inf")))
        e = torch.exp(scores - scores.amax(-1, keepdim=True))  # (a token sees itself)
        out[t:t + step] = torch.matmul(e / e.sum(-1, keepdim=True), v).reshape(-1, H, d).to(q.dtype)
    return s["means"], chosen, out


def _plain_extend(s):
    case, table, lengths = s["case"], s["table"], s["lengths"]
    page, new, pages = case["page"], case["new"], s["k_cache"].shape[0]
    B, width = table.shape
    rows, at = torch.arange(B, device="cuda"), torch.arange(width, device="cuda")
    if s["parents"] is not None:
        parent = s["parents"].long()
        table.copy_(table[parent.clamp(min=0)])
        lengths.copy_(torch.where(parent >= 0, lengths[parent.clamp(min=0)], torch.zeros_like(lengths)))
    held = lengths.long()
    used = (held + page - 1) // page
    entries = torch.where(at < used[:, None], table.long(), torch.full_like(table.long(), -1))
    # Who uses the last page of a row that grows in it?
    rest = held % page
    grows = (rest > 0) & (new > 0)
    last = torch.where(grows, entries[rows, (used - 1).clamp(min=0)], torch.full_like(used, pages))

    def count(ids, ones):
        return torch.zeros(pages + 1, device="cuda", dtype=torch.int64).index_add(0, ids, ones)

    uses = count(torch.where(entries >= 0, entries, torch.full_like(entries, pages)).flatten(),
                 torch.ones(B * width, device="cuda", dtype=torch.int64))
    growing = count(last, torch.ones_like(last))
    lowest = torch.full((pages + 1,), B, device="cuda").scatter_reduce(0, last, rows, "amin")
    copies = grows & ~((uses[last] == growing[last]) & (lowest[last] == rows))
    # The lowest free pages, to the rows in their order.
    free = uses[:pages] == 0
    ids = torch.arange(pages, device="cuda")
    handed = torch.cat([torch.where(free, ids, torch.full_like(ids, pages)).sort().values, ids.new_full((1,), pages)])
    begin = used - copies.long()
    end = torch.clamp((held + new + page - 1) // page, max=width)
    wanted = (end - begin).clamp(min=0)
    first = wanted.cumsum(0) - wanted
    place = (first - begin)[:, None] + at
    fresh = (at >= begin[:, None]) & (at < end[:, None])
    got = handed[place.clamp(0, pages)]
    got = torch.where(got == pages, torch.full_like(got, -1), got)
    table.copy_(torch.where(fresh, got, entries).to(torch.int32))
    # Rows that copy nothing do what the first that does is doing, or write page 0 as it is.
    to = table.long()[rows, (used - 1).clamp(min=0)]
    copies = copies & (to >= 0)
    pick = copies.long().argmax()
    some = copies[pick]
    source = torch.where(copies, last, torch.where(some, last[pick], torch.zeros_like(pick)))
    target = torch.where(copies, to, torch.where(some, to[pick], torch.zeros_like(pick)))
    count_rows = torch.where(copies, rest, torch.where(some, rest[pick], torch.zeros_like(pick)))
    inside = (torch.arange(page, device="cuda") < count_rows[:, None])[:, None]  # (B, 1, page)
    for x in _caches(s):
        x = x.view(torch.uint8) if x.element_size() == 1 else x
        mask = inside[..., None] if x.ndim == 4 else inside
        x[target] = torch.where(mask, x[source], x[target])
    lengths.add_(new)
    return (*_caches(s), table, lengths, (free.sum() - wanted.sum()).to(torch.int32))


def _plain_compact(s):
    page, table = s["case"]["page"], s["table"].long()
    pages, count = s["k_cache"].shape[0], s["num_pages"]
    at = torch.arange(table.shape[1], device="cuda")
    inside = at < ((s["lengths"].long() + page - 1) // page)[:, None]
    ids = torch.where(inside, table, torch.full_like(table, pages))
    used = torch.zeros(pages + 1, device="cuda", dtype=torch.int64).index_fill(0, ids.flatten(), 1)[:pages]
    place = used.cumsum(0) - 1
    order = torch.sort(1 - used, stable=True).indices[:count]
    keep = torch.arange(count, device="cuda") < used.sum()
    got = []
    for x in _caches(s):
        y = x.view(torch.uint8)[order]
        got.append(torch.where(keep.reshape(-1, *[1] * (y.ndim - 1)), y, torch.zeros_like(y)).view(x.dtype))
    ids = torch.where(inside, place[ids.clamp(max=pages - 1)], torch.full_like(ids, -1))
    return (*got, ids.to(torch.int32))


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"rotary": _exact_rotary, "blocks": _exact_blocks, "extend": _exact_extend,
                "compact": _exact_compact}[case["op"]](case, s)


def _turn(case, x, angle):
    """Rows of x (tokens, heads, head_dim) with their pairs, as complex numbers, turned by angle."""
    R, y = case["rotated"], x.clone()
    i = torch.arange(R // 2, device="cuda")
    one, two = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + R // 2)
    z = torch.complex(x[..., one], x[..., two]) * torch.polar(torch.ones_like(angle), angle)[:, None]
    y[..., one], y[..., two] = z.real, z.imag
    return y


def _exact_rotary(case, s):
    h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    tokens = _tokens(case)
    T = int(np.prod(tokens))
    if s["positions"] is not None:
        at = s["positions"].reshape(-1).tolist()
    elif s["lengths"] is not None:
        at = [n - case["n"] + i for n in s["lengths"].tolist() for i in range(case["n"])]
    else:
        at = list(range(case["n"])) * case["batch"]
    angle = torch.tensor(at, dtype=torch.float64, device="cuda")[:, None] * s["frequencies"].double()
    one = {}
    for n, heads in (("q", h), ("k", kv)):
        x = s[n].detach().double().reshape(T, heads, d)
        w = s["w" + n].detach().double() if case["norm"] else torch.ones(d, device="cuda", dtype=torch.float64)
        r = 1 / torch.sqrt((x ** 2).sum(-1, keepdim=True) / d + _EPS) if case["norm"] else torch.ones_like(x[..., :1])
        k3 = r ** 3 / d if case["norm"] else torch.zeros_like(r)  # (the norm's share of the derivatives)
        got = {"y": _turn(case, x * r * w, angle)}
        if case["kind"] != "forward":
            g = _turn(case, s["c" + n].detach().double().reshape(T, heads, d), -angle)
            C = (g * w * x).sum(-1, keepdim=True)
            got["dx"], got["dw"] = r * g * w - k3 * C * x, (g * x * r).sum((0, 1))
        if case["kind"] == "hvp":
            u = s["t" + n].double().reshape(T, heads, d)
            U = (u * x).sum(-1, keepdim=True)
            got["dc"] = r * u * w - k3 * U * w * x
            if case["norm"]:
                z = s["tw" + n].double()
                got["dc"] = got["dc"] + r * z * x
                A, Z = (u * g * w).sum(-1, keepdim=True), (z * g * x).sum(-1, keepdim=True)
                got["dx2"] = -k3 * (x * (A + Z) + g * w * U + C * u) + 3 * k3 * r ** 2 / d * x * C * U + r * z * g
                got["dw2"] = (r * u * g - k3 * U * g * x).sum((0, 1))
            got["dc"] = _turn(case, got["dc"], angle)
        shape = s[n].shape
        one[n] = {k: v if k.startswith("dw") else v.reshape(shape) for k, v in got.items()}
    pick = lambda *names: [one[n][name] for name in names for n in ("q", "k")]
    first = ("dx", "dw") if case["norm"] else ("dx",)
    if case["kind"] == "forward":
        return tuple(pick("y"))
    if case["kind"] == "train":
        return (*pick("y"), *pick(*first))
    return (*pick(*first), *(pick("dx2", "dw2") if case["norm"] else []), *pick("dc"))


def _power(exponent):
    """2 to whole powers in 64 bits, from its bits."""
    return (exponent.to(torch.int64) + 1023 << 52).view(torch.float64)


def _row(s, n, b, length):
    """A sequence's rows of a cache in 64 bits: (length, kv_heads, head_dim)."""
    ids = s["table"][b, :-(-length // s["case"]["page"])].long()
    x = s[n + "_cache"].view(torch.uint8)[ids].view(s[n + "_cache"].dtype).double()
    if s[n + "_scale"] is not None:
        x = x * _power(s[n + "_scale"].view(torch.uint8)[ids].to(torch.int64) - 127)[..., None]
    return x.transpose(1, 2).flatten(0, 1)[:length]


def _exact_blocks(case, s):
    q, page, N = s["q"].double(), case["page"], case["kv_heads"]
    T, H, d = q.shape
    G, most = H // N, case["chosen"]
    means = s["means"].double()
    chosen = torch.full((T, N, most), -1, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(q)
    lengths = s["lengths"].tolist()
    offsets = list(range(T + 1)) if s["offsets"] is None else s["offsets"].tolist()
    for b, length in enumerate(lengths):
        r0, r1 = offsets[b], offsets[b + 1]
        n = r1 - r0
        k, v = _row(s, "k", b, length), _row(s, "v", b, length)
        ids = s["table"][b].long()
        for j in range((length - n) // page, length // page):  # (a mean is held in 32 bits)
            means[ids[j]] = (k[j * page:(j + 1) * page].sum(0) / page).float().double()
        pos = torch.arange(length - n, length, device="cuda")
        at = pos // page
        count = -(-length // page)
        j = torch.arange(count, device="cuda")
        seen = torch.arange(length, device="cuda") <= pos[:, None]
        for h in range(N):
            sums = q[r0:r1, h * G:(h + 1) * G].sum(1)
            score = sums @ means[ids[:count], h].T
            free = (j >= case["first"]) & (j <= (at - case["last"])[:, None])
            forced = (j <= at[:, None]) & ~free
            room = torch.clamp(most - forced.sum(-1, keepdim=True), min=0)
            # how many free pages come before a page: a larger score, or as large and a lower index
            by = torch.sort(score.masked_fill(~free, float("-inf")), dim=-1, descending=True, stable=True).indices
            place = torch.empty_like(by).scatter_(-1, by, j.expand_as(by).contiguous())
            takes = forced | (free & (place < room))
            index = torch.where(takes, j, count).sort(-1).values[:, :most]
            chosen[r0:r1, h, :index.shape[1]] = torch.where(index < count, index, -1).to(torch.int32)
            mask = seen & takes.repeat_interleave(page, -1)[:, :length]
            for g in range(h * G, (h + 1) * G):
                x = ((q[r0:r1, g] @ k[:, h].T) * d ** -0.5).masked_fill(~mask, float("-inf"))
                out[r0:r1, g] = torch.softmax(x, -1) @ v[:, h].contiguous()
    return means, chosen, out


def _exact_extend(case, s):
    """The definition, one row and page after the other."""
    page, new = case["page"], case["new"]
    table, lengths = s["table"].tolist(), s["start"].tolist()
    width, pages = len(table[0]), s["k_cache"].shape[0]
    if s["parents"] is not None:
        parents = s["parents"].tolist()
        table, lengths = [list(table[p]) for p in parents], [lengths[p] for p in parents]
    used = [-(-n // page) for n in lengths]
    users = {}
    for b, n in enumerate(used):
        for c in range(n):
            users.setdefault(table[b][c], []).append(b)
    growing = {}
    for b, n in enumerate(lengths):
        if n % page and new:
            growing.setdefault(table[b][used[b] - 1], []).append(b)
    free = [i for i in range(pages) if i not in users]
    left, copies = len(free), []
    free = iter(free)
    for b, n in enumerate(lengths):
        begin = used[b]
        if n % page and new:
            last = table[b][begin - 1]
            if len(users[last]) > len(growing[last]) or growing[last][0] != b:
                begin -= 1
                copies.append((b, last, n % page))
        end = min(width, -(-(n + new) // page))
        for c in range(begin, end):
            table[b][c] = next(free, -1)
        left -= max(0, end - begin)
        for c in range(max(end, used[b]), width):
            table[b][c] = -1
    got = [x.to(torch.float32).double() if x.dtype != torch.float8_e8m0fnu
           else _power(x.view(torch.uint8).to(torch.int64) - 127) for x in _caches(s)]
    for b, source, rows in copies:
        target = table[b][used[b] - 1]
        if target >= 0:
            for x in got:
                x[target, :, :rows] = x[source, :, :rows]
    return (*got, torch.tensor(table, dtype=torch.int32, device="cuda"),
            torch.tensor([n + new for n in lengths], dtype=torch.int32, device="cuda"),
            torch.tensor(left, dtype=torch.int32, device="cuda"))


def _exact_compact(case, s):
    page = case["page"]
    table, lengths = s["table"].tolist(), s["lengths"].tolist()
    used = sorted({table[b][c] for b, n in enumerate(lengths) for c in range(-(-n // page))})
    place = {old: i for i, old in enumerate(used)}
    table = [[place[x] if c < -(-n // page) else -1 for c, x in enumerate(row)] for row, n in zip(table, lengths)]
    # Copies are no computed numbers; a small cache's are given all the same.
    got = [None] * len(_caches(s))
    if s["k_cache"].numel() < 2 ** 24:
        ids = torch.tensor(used, device="cuda", dtype=torch.int64)
        for i, x in enumerate(_caches(s)):
            picked = x.view(torch.uint8)[ids].view(x.dtype)
            values = (_power(picked.view(torch.uint8).to(torch.int64) - 127) if x.dtype == torch.float8_e8m0fnu
                      else picked.to(torch.float32).double())
            # (the pages behind are zero bytes)
            rest = torch.full((s["num_pages"] - len(used), *values.shape[1:]),
                              2.0 ** -127 if x.dtype == torch.float8_e8m0fnu else 0.0, dtype=torch.float64, device="cuda")
            got[i] = torch.cat([values, rest])
    return (*got, torch.tensor(table, dtype=torch.int32, device="cuda"))
