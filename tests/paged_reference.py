"""A paged cache and its operators in plain 64-bit torch on the CPU, one sequence and head at a
time: the oracle of the paged kernels' tests."""

from __future__ import annotations

import torch

E4M3 = torch.float8_e4m3fn


def powers(code):
    """2^(code - 127) of e8m0 bytes, in 64 bits."""
    return torch.ldexp(torch.ones((), dtype=torch.float64), code.to(torch.int64) - 127)


def quantise(x):
    """e4m3 codes (bytes) and e8m0 scale bytes of the rows of x, from the definition: the smallest
    power of two s >= 2^-126 with max |x| / s <= 448 (finite magnitudes), then x / s to nearest even."""
    x = x.double()
    finite = torch.isfinite(x)
    amax = torch.where(finite, x.abs(), torch.zeros_like(x)).amax(-1)
    code = torch.ones(amax.shape, dtype=torch.int64)
    for c in range(2, 255):
        code = torch.where(448 * powers(torch.tensor(c - 1)) < amax, c, code)
    y = torch.where(finite, x / powers(code)[..., None], torch.full_like(x, float("nan")))
    return y.float().to(E4M3).view(torch.uint8), code.to(torch.uint8)


class Cache:
    """A cache that holds `lengths` tokens of random keys and values, NaN (or 0x7f) everywhere
    else, sequences' pages in random order and -1 in the table where no page is."""

    def __init__(self, lengths, page, kv_heads, head_dim, dtype, quantised, seed=0, spare=2, width=None):
        gen = torch.Generator().manual_seed(seed)
        used = [-(-n // page) for n in lengths]
        pages = sum(used) + spare
        width = max(used + [1]) + 1 if width is None else width
        ids = torch.randperm(pages, generator=gen).tolist()
        self.table = torch.full((len(lengths), width), -1, dtype=torch.int32)
        for b, n in enumerate(used):
            for j in range(n):
                self.table[b, j] = ids.pop()
        self.lengths, self.page, self.dtype = list(lengths), page, dtype
        shape = (pages, kv_heads, page, head_dim)
        self.dense, self.cache, self.scale = {}, {}, {}
        for n in "kv":
            rows = torch.randn(shape, generator=gen) * torch.exp(0.5 * torch.randn(shape[:3] + (1,), generator=gen))
            rows = rows.to(dtype)
            if quantised:
                codes, scale = quantise(rows)
            for b, length in enumerate(lengths):  # what no token has written
                if length % page:
                    last = int(self.table[b, used[b] - 1])
                    rows[last, :, length % page:] = float("nan")
                    if quantised:
                        codes[last, :, length % page:] = 0x7F
            for j in ids:
                rows[j] = float("nan")
                if quantised:
                    codes[j] = 0x7F
            self.cache[n] = codes.view(E4M3) if quantised else rows
            self.scale[n] = scale if quantised else None

    def rows(self, n, b, length):
        """Keys or values of a sequence's first `length` tokens, (length, kv_heads, head_dim), 64 bits."""
        ids = self.table[b, :-(-length // self.page)].long()
        x = self.cache[n].view(torch.uint8)[ids].view(E4M3).double() if self.scale[n] is not None \
            else self.cache[n][ids].double()
        if self.scale[n] is not None:
            x = x * powers(self.scale[n][ids])[..., None]
        return x.transpose(1, 2).flatten(0, 1)[:length]

    def on(self, device):
        """Keyword arguments of the operators."""
        moved = {"key_cache": self.cache["k"].to(device), "value_cache": self.cache["v"].to(device),
                 "page_table": self.table.to(device),
                 "lengths": torch.tensor(self.lengths, dtype=torch.int32, device=device)}
        if self.scale["k"] is not None:
            moved["key_scale"] = self.scale["k"].to(device).view(torch.float8_e8m0fnu)
            moved["value_scale"] = self.scale["v"].to(device).view(torch.float8_e8m0fnu)
        return moved


def attention(q, cache, new, window, sinks, scale):
    """Outputs of the packed new tokens q, `new[b]` of sequence b, in 64 bits."""
    q = q.double()
    out = torch.zeros_like(q)
    group = q.shape[1] // cache.cache["k"].shape[1]
    row = 0
    for b, (count, length) in enumerate(zip(new, cache.lengths)):
        k, v = cache.rows("k", b, length), cache.rows("v", b, length)
        for i in range(count):
            p = length - count + i
            s = torch.arange(max(0, p + 1))
            seen = s[(s > p - window) | (s < sinks)] if window else s
            for h in range(q.shape[1]):
                if len(seen):
                    w = torch.softmax(k[seen, h // group] @ q[row, h] * scale, 0)
                    out[row, h] = w @ v[seen, h // group]
            row += 1
    return out
