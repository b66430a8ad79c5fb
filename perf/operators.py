"""Windowed attention and the paged key/value cache: performance cases of their operators.

listed() names the cases, draw(rng) gives one more of the same ranges, prepare(case, seed)
makes the inputs on the GPU, run(state) is one pass, work(case) its least bytes and flops,
exact(case, seed) the outputs in 64 bits.

The operators (`op`):

  window  dot_product_attention(..., window=W, sinks=S): causal attention in which a query at
          position p sees the keys p - W < s <= p and, besides, the first S keys (s < S).
          `kind` forward: no autograd; train: with the gradients of q, k, v for an upstream
          gradient; hvp: the gradients and their derivative along tangents of q, k, v.
  paged   paged_attention: packed new tokens of several sequences against the keys that a page
          table finds in a cache, one token per sequence (`new` = 1) or a chunk of them.
  write   paged_cache_write: the keys and values of new tokens into their sequences' pages,
          quantised on the way where the cache holds e4m3.
  read    paged_cache_read: the keys and values of the sequences back as dense tensors.

A cache is (pages, kv_heads, page_size, head_dim); an e4m3 cache has an e8m0 scale (a power of
two) for each key and value row, (pages, kv_heads, page_size): the smallest with which the
row's largest magnitude stays within e4m3's 448.
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


def _window(name, kind, batch, n_q, n_k, heads, kv_heads, head_dim, dtype, alignment, window, sinks):
    case = {"op": "window", "kind": kind, "batch": batch, "n_q": n_q, "n_k": n_k, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "alignment": alignment, "window": window,
            "sinks": sinks}
    return {"name": name, **case} if name else case


def _cache(name, op, batch, new_min, new, length_min, length, heads, kv_heads, head_dim, dtype, cache, page, window=0,
           sinks=0):
    """`new` tokens at most (new_min at least) in each of `batch` sequences that hold length_min
    to `length` tokens with the new ones; window 0: none."""
    case = {"op": op, "batch": batch, "new_min": new_min, "new": new, "length_min": length_min, "length": length,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "cache": cache, "page": page,
            "window": window, "sinks": sinks}
    return {"name": name, **case} if name else case


def listed():
    return [
        # Inference on one short sequence: launches and host time weigh most.
        _window("window_forward_b1_n300_h12_d64", "forward", 1, 300, 300, 12, 12, 64, "bf16", "top_left", 128, 4),
        # A training step in full precision against a longer context that is given (as a second-order
        # method's accuracy reference runs), no size a multiple of a tile.
        _window("window_train_b1_q1000_k1333_h8_d64_fp32", "train", 1, 1000, 1333, 8, 8, 64, "fp32", "bottom_right",
                256, 16),
        # A training step with grouped heads, 128 wide, ragged, no sinks.
        _window("window_train_b2_n4001_h32_kv8_d128_fp16", "train", 2, 4001, 4001, 32, 8, 128, "fp16", "top_left",
                1024, 0),
        # A curvature probe on one long sequence: what a window is for.
        _window("window_hvp_b1_n16384_h12_d64", "hvp", 1, 16384, 16384, 12, 12, 64, "bf16", "top_left", 1024, 4),
        # The next token of one conversation: latency.
        _cache("paged_token_b1_len1000_h16_kv4_d64", "paged", 1, 1, 1, 1000, 1000, 16, 4, 64, "bf16", "bf16", 16),
        # The next token of a batch of long, unequal conversations over a quantised cache.
        _cache("paged_token_b16_len32768_h32_kv8_d128_e4m3", "paged", 16, 1, 1, 2000, 32768, 32, 8, 128, "bf16",
               "e4m3", 64),
        # Short and longer pieces of prompts together, on contexts of unequal length, with a window
        # and sinks.
        _cache("paged_chunk_b8_new512_len8192_h32_kv8_d128_window", "paged", 8, 17, 512, 700, 8192, 32, 8, 128, "bf16",
               "bf16", 16, 2048, 4),
        # A long prompt's last quarter over a quantised cache, without grouping.
        _cache("paged_chunk_b1_new4096_len16384_h12_d64_fp16_e4m3", "paged", 1, 4096, 4096, 16384, 16384, 12, 12, 64,
               "fp16", "e4m3", 64),
        # One new token of each sequence of a batch enters its page.
        _cache("write_b64_new1_kv8_d128_e4m3", "write", 64, 1, 1, 1, 8192, 8, 8, 128, "bf16", "e4m3", 64),
        # Prompts enter the cache.
        _cache("write_b4_new8192_kv16_d64_e4m3", "write", 4, 5001, 8192, 5001, 8192, 16, 16, 64, "bf16", "e4m3", 64),
        # A short cached prefix comes back as dense tensors (to score or train on it).
        _cache("read_b1_len500_kv4_d64", "read", 1, 1, 1, 500, 500, 4, 4, 64, "bf16", "bf16", 16),
        # A batch of long cached sequences comes back.
        _cache("read_b8_len16384_kv8_d128_e4m3", "read", 8, 1, 1, 3001, 16384, 8, 8, 128, "bf16", "e4m3", 64),
    ]


# ------------------------------------------------------------------ more cases

def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_window(rng):
    kind = rng.choice(("forward", "train", "hvp"))
    dtype = rng.choices(("bf16", "fp16", "fp32"), (5, 3, 2))[0]
    n_q = _log_int(rng, 1 if kind == "forward" else 16, 16384)
    alignment = rng.choice(("top_left", "top_left", "bottom_right"))
    n_k = n_q if alignment == "top_left" else max(1, int(n_q * rng.uniform(0.7, 2.5)))
    kv_heads = rng.choice((1, 2, 4, 8, 12, 16))
    return _window(None, kind, _log_int(rng, 1, 32), n_q, n_k, kv_heads * rng.choice((1, 1, 2, 4)), kv_heads,
                   rng.choice((64, 128) if dtype == "fp32" else (64, 64, 128, 128, 256)), dtype, alignment,
                   _log_int(rng, 16, 4096), rng.choice((0, 1, 4, 4, 16, 100)))


def _draw_cache(rng):
    op = rng.choice(("paged", "paged", "write", "read"))
    batch = _log_int(rng, 1, 64)
    length = _log_int(rng, 16, 32768)
    length_min = max(1, int(length * rng.uniform(0.1, 1.0)))
    new = 1 if op == "read" or rng.random() < 0.5 else min(length_min, _log_int(rng, 2, 8192))
    new_min = max(1, int(new * rng.uniform(0.1, 1.0)))
    kv_heads = rng.choice((1, 2, 4, 8, 12, 16))
    heads = kv_heads * (rng.choice((1, 1, 2, 4, 8)) if op == "paged" else 1)
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    window, sinks = (_log_int(rng, 16, 8192), rng.choice((0, 1, 4, 16))) if op == "paged" and rng.random() < 0.4 else (0, 0)
    return _cache(None, op, batch, new_min, new, length_min, length, heads, kv_heads, rng.choice((64, 128, 128, 256)),
                  dtype, rng.choice((dtype, "e4m3")), rng.choice((16, 16, 32, 64, 128, 256)), window, sinks)


def draw(rng):
    """One case of the ranges above: 1 to 16384 queries and 1 to 2.5 times as many keys, or 16 to
    32768 cached tokens (sizes over their logarithm, odd ones among them), 1 to 64 sequences, 1 to
    64 heads, grouped or not, each dtype, head dim, page size, window and kind."""
    biggest = {}
    for case in listed():
        w = work(case)
        best = biggest.setdefault(case["op"], {"bytes": 0, "flops": 0, "plain": 0})
        for key, value in {**w, "plain": _plain_values(case)}.items():
            best[key] = max(best[key], value)
    while True:
        case = _draw_window(rng) if rng.random() < 0.45 else _draw_cache(rng)
        most = biggest[case["op"]]
        if case["heads"] <= 64 and all(v <= most[key] for key, v in {**work(case), "plain": _plain_values(case)}.items()):
            return case


def _plain_values(case):
    """Numbers in the plain form's largest tensor."""
    if case["op"] == "window":
        positions, block = _blocks(case)
        return case["batch"] * case["heads"] * positions * (2 * block + case["sinks"])
    per_token = {"paged": case["heads"] * case["new"] + case["kv_heads"] * case["head_dim"],
                 "write": case["kv_heads"] * case["head_dim"], "read": case["kv_heads"] * case["head_dim"]}[case["op"]]
    return case["batch"] * case["length"] * per_token


# ------------------------------------------------------------------ sizes that a case implies

def _off(case):
    """Position of the first query."""
    return case["n_k"] - case["n_q"] if case["alignment"] == "bottom_right" else 0


def _visible(p, n_k, window, sinks):
    """How many of n_k keys a query at each position p sees, and the first key of its window."""
    hi = np.clip(p + 1, 0, n_k)
    lo = np.clip(p + 1 - window, 0, n_k) if window else np.zeros_like(p)
    return np.maximum(hi - lo, 0) + np.minimum(sinks, np.minimum(lo, hi)), lo


def _spread(lo, hi, count):
    """`count` whole numbers from hi down to lo."""
    return np.array([hi if count == 1 else hi - (hi - lo) * i // (count - 1) for i in range(count)])


def _counts(case):
    """New tokens and lengths of the sequences, before a seed puts them in an order."""
    return _spread(case["new_min"], case["new"], case["batch"]), _spread(case["length_min"], case["length"], case["batch"])


def _pages_per_sequence(case):
    return -(-case["length"] // case["page"]) + 1


def work(case):
    d, item = case["head_dim"], _BYTES[case["dtype"]]
    if case["op"] == "window":
        p = np.arange(case["n_q"], dtype=np.int64) + _off(case)
        pairs = int(_visible(p, case["n_k"], case["window"], case["sinks"])[0].sum()) * case["batch"] * case["heads"]
        q = case["batch"] * case["n_q"] * case["heads"] * d * item
        k = case["batch"] * case["n_k"] * case["kv_heads"] * d * item
        products, size = {
            "forward": (2, 2 * q + 2 * k),   # q k v -> out
            "train": (7, 4 * q + 4 * k),     # q k v cot -> out dq dk dv
            "hvp": (19, 5 * q + 8 * k),      # q k v cot tangents -> gradients, products
        }[case["kind"]]
        return {"bytes": size, "flops": products * 2 * d * pairs}
    new, lengths = _counts(case)
    row = 2 * (d * _BYTES[case["cache"]] + (1 if case["cache"] == "e4m3" else 0))  # a token's key and value of a head
    dense = 2 * d * item
    table = 4 * case["batch"] * _pages_per_sequence(case)
    if case["op"] == "write":
        return {"bytes": int(new.sum()) * case["kv_heads"] * (dense + row), "flops": 2 * int(new.sum()) * case["kv_heads"] * d}
    if case["op"] == "read":
        return {"bytes": case["kv_heads"] * (int(lengths.sum()) * row + case["batch"] * case["length"] * dense) + table,
                "flops": 2 * int(lengths.sum()) * case["kv_heads"] * d}
    pairs, keys = 0, 0
    for count, length in zip(new, lengths):
        p = np.arange(length - count, length, dtype=np.int64)
        seen, lo = _visible(p, int(length), case["window"], case["sinks"])
        pairs += int(seen.sum())
        keys += int(length - lo[0]) + min(case["sinks"], int(lo[0]))
    return {"bytes": keys * case["kv_heads"] * row + int(new.sum()) * case["heads"] * dense + table,
            "flops": 4 * d * pairs * case["heads"]}


# ------------------------------------------------------------------ inputs

def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _exponent(amax):
    """The e8m0 code of each row's scale from its largest magnitude (fp32): 2^(code - 127)."""
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa 2^exponent, mantissa in [1/2, 1)
    code = exponent - 1 - 8 + (mantissa > 0.875).to(exponent.dtype) + 127
    return torch.where(amax > 0, code, torch.ones_like(code)).clamp(1, 254).to(torch.uint8)


def _scales(code):
    """The powers of two that e8m0 codes (bytes, 1 to 254) stand for, in fp32: the exponent's bits, as
    exp2 and pow need not be exact."""
    return (code.to(torch.int32) << 23).view(torch.float32)


def _quantise(x):
    """e4m3 values and e8m0 scales of the rows of x (their last axis), as bytes."""
    x = x.float()
    code = _exponent(x.abs().amax(-1))
    return (x / _scales(code)[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), code


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "window":
        q_shape = (case["batch"], case["n_q"], case["heads"], case["head_dim"])
        k_shape = (case["batch"], case["n_k"], case["kv_heads"], case["head_dim"])
        names = {"forward": ("q", "k", "v"), "train": ("q", "k", "v", "cot"),
                 "hvp": ("q", "k", "v", "cot", "tq", "tk", "tv")}[case["kind"]]
        x = {n: _normal(gen, q_shape if n in ("q", "cot", "tq") else k_shape, dtype) for n in names}
        if case["kind"] != "forward":
            for n in ("q", "k", "v"):
                x[n].requires_grad_()
        return {"case": case, **x}
    batch, page, kv, d = case["batch"], case["page"], case["kv_heads"], case["head_dim"]
    order = np.random.RandomState(seed)
    new, lengths = _counts(case)
    at = order.permutation(batch)  # which sequence is how long has nothing to do with its place
    new, lengths = new[at], lengths[at]
    width = _pages_per_sequence(case)
    used = -(-lengths // page)
    pages = int(used.sum()) + 3
    table = np.full((batch, width), -1, dtype=np.int32)  # no page behind a sequence's last
    ids, first = order.permutation(pages), 0
    for b in range(batch):
        table[b, :used[b]] = ids[first:first + used[b]]
        first += used[b]
    state = {"case": case, "table": torch.from_numpy(table).cuda(),
             "lengths": torch.from_numpy(lengths.astype(np.int32)).cuda(), "offsets": None}
    if case["new"] > 1:
        state["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).cuda()
    total = int(new.sum())
    # rows of unlike magnitude, as keys and values have them
    for n in ("k", "v"):
        rows = torch.randn((pages, kv, page, d), generator=gen, device="cuda")
        rows *= torch.exp(0.5 * torch.randn((pages, kv, page, 1), generator=gen, device="cuda")) * 0.7
        if case["cache"] == "e4m3":
            values, code = _quantise(rows)
            state[n + "_cache"] = values.view(torch.float8_e4m3fn)
            state[n + "_scale"] = code.view(torch.float8_e8m0fnu)
        else:
            state[n + "_cache"], state[n + "_scale"] = rows.to(dtype), None
        del rows
    if case["op"] == "paged":
        state["q"] = _normal(gen, (total, case["heads"], d), dtype)
        # slots that hold no token yet may hold anything
        slot = torch.arange(page, device="cuda")
        for b in np.flatnonzero(lengths % page):
            last = int(table[b, used[b] - 1])
            empty = slot >= int(lengths[b] % page)
            for n in ("k", "v"):
                if case["cache"] == "e4m3":
                    state[n + "_cache"].view(torch.uint8)[last, :, empty] = 0x7F
                else:
                    state[n + "_cache"][last, :, empty] = float("nan")
    elif case["op"] == "write":
        for n in ("k", "v"):
            state[n] = (torch.randn((total, kv, d), generator=gen, device="cuda")
                        * torch.exp(0.5 * torch.randn((total, kv, 1), generator=gen, device="cuda"))).to(dtype)
    return state


# ------------------------------------------------------------------ one pass

def run(s):
    case = s["case"]
    if case["op"] == "window":
        leaves = (s["q"], s["k"], s["v"])
        if case["kind"] == "forward":
            with torch.no_grad():
                return _window_attention(s, *leaves)
        out = _window_attention(s, *leaves)
        if case["kind"] == "train":
            return (out.detach(), *torch.autograd.grad(out, leaves, s["cot"]))
        grads = torch.autograd.grad(out, leaves, s["cot"], create_graph=True)
        products = torch.autograd.grad(grads, leaves, (s["tq"], s["tk"], s["tv"]))
        return (*(g.detach() for g in grads), *products)
    if own:
        return _call(s)
    return {"paged": _plain_paged, "write": _plain_write, "read": _plain_read}[case["op"]](s)


def _window_attention(s, q, k, v):
    case = s["case"]
    if own:
        return _flash_hog().dot_product_attention(q, k, v, True, causal_alignment=case["alignment"],
                                                  window=case["window"], sinks=case["sinks"])
    return _plain_window(case, q, k, v)


def _flash_hog():
    if _PACKAGE_ROOT not in sys.path:
        sys.path.insert(0, _PACKAGE_ROOT)
    import flash_hog

    return flash_hog


def _call(s):
    case, hog = s["case"], _flash_hog()
    scales = {"key_scale": s["k_scale"], "value_scale": s["v_scale"]}
    if case["op"] == "paged":
        return hog.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["offsets"],
                                   window=case["window"] or None, sinks=case["sinks"], **scales)
    if case["op"] == "write":
        hog.paged_cache_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lengths"], s["offsets"],
                              **scales)
        return _caches(s)
    return hog.paged_cache_read(s["k_cache"], s["v_cache"], s["table"], s["lengths"], max_length=case["length"],
                                dtype=_DTYPES[case["dtype"]], **scales)


def _caches(s):
    return tuple(s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale") if s[n] is not None)


# ------------------------------------------------------------------ plain forms

def _softmax(scores, mask):
    """Softmax over the last axis of the scores where mask; zeros in rows with none."""
    scores = torch.where(mask, scores, torch.full_like(scores, float("-inf")))
    top = scores.detach().amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, torch.ones_like(total))


def _blocks(case):
    """Positions of queries and keys, padded to whole blocks, and a block: the window, or all."""
    positions = max(case["n_k"], case["n_q"] + _off(case), 1)
    block = min(case["window"], positions)
    return -(-positions // block) * block, block


def _plain_window(case, q, k, v):
    """Queries in blocks of the window's size, each against its own block of keys, the one before
    it and the sinks."""
    B, n_q, H, d = q.shape
    n_k, N, off, S = case["n_k"], case["kv_heads"], _off(case), min(case["sinks"], case["n_k"])
    G, dtype = H // N, q.dtype
    P, W = _blocks(case)
    nb = P // W
    skip = max(0, -off)  # queries before the first key
    first = max(0, off)  # position of the first query kept

    def zeros(x, rows):
        return torch.zeros((B, rows, *x.shape[2:]), device=x.device, dtype=torch.float32)

    qf = q[:, skip:].float()
    qf = torch.cat([zeros(qf, first), qf, zeros(qf, P - first - qf.shape[1])], 1)
    qf = qf.reshape(B, nb, W, N, G, d).permute(0, 3, 1, 4, 2, 5).reshape(B, N, nb, G * W, d)

    def banded(x):
        x = x.float()
        sink = x[:, :S].permute(0, 2, 1, 3)[:, :, None].expand(B, N, nb, S, d)
        x = torch.cat([zeros(x, W), x, zeros(x, P - n_k)], 1)
        x = x.reshape(B, nb + 1, W, N, d).permute(0, 3, 1, 2, 4)
        return torch.cat([sink, x[:, :, :-1], x[:, :, 1:]], 3)  # (B, N, nb, S + 2 W, d)

    kf, vf = banded(k), banded(v)
    t = torch.arange(W, device=q.device)
    start = torch.arange(nb, device=q.device)[:, None, None] * W
    pos = start + t[None, :, None]  # (nb, W, 1)
    key = start - W + torch.arange(2 * W, device=q.device)  # (nb, 1, 2 W)
    band = (key >= 0) & (key < n_k) & (key <= pos) & (key > pos - case["window"])
    sink = torch.arange(S, device=q.device)
    mask = torch.cat([(sink <= pos - case["window"]).expand(nb, W, S), band], 2)  # sinks that the window lacks
    scores = torch.matmul(qf, kf.transpose(-1, -2)) * d ** -0.5
    w = _softmax(scores.reshape(B, N, nb, G, W, S + 2 * W), mask[:, None])
    out = torch.matmul(w.reshape(B, N, nb, G * W, S + 2 * W), vf)
    out = out.reshape(B, N, nb, G, W, d).permute(0, 2, 4, 1, 3, 5).reshape(B, P, H, d)
    out = out[:, first:first + n_q - skip]
    return torch.cat([zeros(out, skip), out], 1).to(dtype)


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


def _gathered(s, n):
    """The sequences' rows of a cache, dequantised: (batch, kv_heads, tokens, head_dim) in fp32."""
    table = s["table"].clamp(min=0).long()
    x = s[n + "_cache"].view(torch.uint8)[table].view(s[n + "_cache"].dtype).float()
    if s[n + "_scale"] is not None:
        x = x * _scales(s[n + "_scale"].view(torch.uint8)[table])[..., None]
    B, P, N, page, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, N, P * page, d)


def _plain_paged(s):
    case, q = s["case"], s["q"]
    T, H, d = q.shape
    N = case["kv_heads"]
    G, new = H // N, case["new"]
    row_b, row_i, counts, starts = _sequence_rows(s, T)
    k, v = _gathered(s, "k"), _gathered(s, "v")
    B, _, L, _ = k.shape
    lengths = s["lengths"].long()
    key = torch.arange(L, device="cuda")
    v = torch.where((key < lengths[:, None])[:, None, :, None], v, torch.zeros_like(v))
    i = torch.arange(new, device="cuda")
    qp = q[(starts[:, None] + i).clamp(max=T - 1)].float()  # (B, new, H, d), some rows of the next sequence's
    qp = qp.reshape(B, new, N, G, d).permute(0, 2, 3, 1, 4).reshape(B, N, G * new, d)
    pos = (lengths - counts)[:, None, None] + i[:, None]  # (B, new, 1)
    mask = key <= pos.clamp(max=lengths[:, None, None] - 1)
    if case["window"]:
        mask = mask & ((key > pos - case["window"]) | (key < case["sinks"]))
    scores = torch.matmul(qp, k.transpose(-1, -2)).reshape(B, N, G, new, L) * d ** -0.5
    w = _softmax(scores, mask[:, None, None])
    out = torch.matmul(w.reshape(B, N, G * new, L), v)
    out = out.reshape(B, N, G, new, d).permute(0, 3, 1, 2, 4).reshape(B, new, H, d)
    return out[row_b, row_i].to(q.dtype)


def _plain_write(s):
    page = s["case"]["page"]
    b, i, counts, _ = _sequence_rows(s, s["k"].shape[0])
    pos = s["lengths"].long()[b] - counts[b] + i
    at = s["table"].long()[b, pos // page]
    for n in ("k", "v"):
        if s[n + "_scale"] is None:
            s[n + "_cache"][at, :, pos % page] = s[n]
        else:
            values, code = _quantise(s[n])
            s[n + "_cache"].view(torch.uint8)[at, :, pos % page] = values
            s[n + "_scale"].view(torch.uint8)[at, :, pos % page] = code
    return _caches(s)


def _plain_read(s):
    case = s["case"]
    length, got = case["length"], []
    valid = torch.arange(length, device="cuda") < s["lengths"][:, None]
    for n in ("k", "v"):
        x = _gathered(s, n)[:, :, :length].permute(0, 2, 1, 3)
        got.append(torch.where(valid[:, :, None, None], x, torch.zeros_like(x)).to(_DTYPES[case["dtype"]]))
    return tuple(got)


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"window": _exact_window, "paged": _exact_paged, "write": _exact_write, "read": _exact_read}[case["op"]](case, s)


def _attend(q, k, v, pos, window, sinks, scale):
    """One head's outputs (queries at positions pos, keys from 0 on) from the whole score matrix."""
    s = torch.arange(k.shape[0], device="cuda")[None, :]
    hidden = s > pos[:, None]
    if window:
        hidden = hidden | ((s <= pos[:, None] - window) & (s >= sinks))
    x = ((q @ k.T) * scale).masked_fill(hidden, -1e300)
    x = torch.exp(x - x.amax(-1, keepdim=True).detach()).masked_fill(hidden, 0.0)
    total = x.sum(-1, keepdim=True)
    return (x @ v) / total.masked_fill(total == 0, 1.0)


def _exact_window(case, s):
    names = [n for n in ("q", "k", "v", "cot", "tq", "tk", "tv") if n in s]
    x = {n: s[n].detach().double() for n in names}
    pos = torch.arange(case["n_q"], device="cuda") + _off(case)
    G = case["heads"] // case["kv_heads"]
    out = torch.zeros_like(x["q"])
    sums = {n: [torch.zeros_like(x[n]) for _ in range(2)] for n in ("q", "k", "v")}
    for b in range(case["batch"]):
        for h in range(case["heads"]):
            g = h // G
            one = {n: x[n][b, :, h if n in ("q", "cot", "tq") else g].clone() for n in names}
            leaves = [one[n].requires_grad_(case["kind"] != "forward") for n in ("q", "k", "v")]
            o = _attend(*leaves, pos, case["window"], case["sinks"], case["head_dim"] ** -0.5)
            out[b, :, h] = o.detach()
            if case["kind"] == "forward":
                continue
            first = torch.autograd.grad(o, leaves, one["cot"], create_graph=case["kind"] == "hvp")
            both = [first]
            if case["kind"] == "hvp":
                both.append(torch.autograd.grad(first, leaves, [one["tq"], one["tk"], one["tv"]]))
            for which, grads in enumerate(both):
                for n, y in zip(("q", "k", "v"), grads):
                    sums[n][which][b, :, h if n == "q" else g] += y.detach()
    if case["kind"] == "forward":
        return out
    grads = tuple(sums[n][0] for n in ("q", "k", "v"))
    return (out, *grads) if case["kind"] == "train" else (*grads, *(sums[n][1] for n in ("q", "k", "v")))


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


def _new_rows(s):
    """(sequence, its length, first and last packed row) of each sequence."""
    lengths = s["lengths"].tolist()
    offsets = range(len(lengths) + 1) if s["offsets"] is None else s["offsets"].tolist()
    return [(b, n, offsets[b], offsets[b + 1]) for b, n in enumerate(lengths)]


def _exact_paged(case, s):
    q = s["q"].double()
    out = torch.zeros_like(q)
    G = case["heads"] // case["kv_heads"]
    for b, length, r0, r1 in _new_rows(s):
        k, v = _row(s, "k", b, length), _row(s, "v", b, length)
        pos = torch.arange(length - (r1 - r0), length, device="cuda")
        for h in range(case["heads"]):
            out[r0:r1, h] = _attend(q[r0:r1, h], k[:, h // G].contiguous(), v[:, h // G].contiguous(), pos,
                                    case["window"], case["sinks"], case["head_dim"] ** -0.5)
    return out


def _exact_write(case, s):
    got = {n: s[n].double() if s[n].dtype != torch.float8_e8m0fnu else _power(s[n].view(torch.uint8).to(torch.int64) - 127)
           for n in ("k_cache", "v_cache", "k_scale", "v_scale") if s[n] is not None}
    for b, length, r0, r1 in _new_rows(s):
        pos = torch.arange(length - (r1 - r0), length, device="cuda")
        at = s["table"][b].long()[pos // case["page"]]
        for n in ("k", "v"):
            x = s[n][r0:r1].double()
            if case["cache"] == "e4m3":
                amax = x.abs().amax(-1).clamp(min=448 * 2.0 ** -126)
                power = torch.round(torch.log2(amax / 448))  # and then the smallest power of two that will do
                power = torch.where(_power(power) * 448 < amax, power + 1, power)
                power = torch.where(_power(power - 1) * 448 >= amax, power - 1, power)
                got[n + "_scale"][at, :, pos % case["page"]] = _power(power)
                x = x / _power(power)[..., None]
                step = _power(torch.frexp(x.abs().clamp(min=2.0 ** -6))[1] - 1 - 3)  # of e4m3 around x
                x = torch.round(x / step) * step
            got[n + "_cache"][at, :, pos % case["page"]] = x
    return tuple(got.values())


def _exact_read(case, s):
    shape = (case["batch"], case["length"], case["kv_heads"], case["head_dim"])
    got = tuple(torch.zeros(shape, device="cuda", dtype=torch.float64) for _ in range(2))
    for b, length, _, _ in _new_rows(s):
        for n, out in zip(("k", "v"), got):
            out[b, :length] = _row(s, n, b, length)
    return got
