"""Attention over chosen blocks in plain 64-bit torch on the CPU, one token and head at a time: the
oracle of its kernels' tests. Caches are paged_reference.Cache."""

from __future__ import annotations

import torch


def key_means(cache, new, means):
    """means (pages, kv_heads, head_dim) fp32 with those of the pages that the last new[b] tokens fill."""
    means, page = means.clone(), cache.page
    for b, (count, length) in enumerate(zip(new, cache.lengths)):
        keys = cache.rows("k", b, length)
        for j in range(max(0, length - count) // page, length // page):
            means[cache.table[b, j].long()] = (keys[j * page:(j + 1) * page].sum(0) / page).float()
    return means


def select(q, means, table, lengths, new, page, blocks, first, last):
    """Columns that each packed token attends to, (T, kv_heads, blocks), -1 behind them."""
    T, H, _ = q.shape
    pages, N, _ = means.shape
    q, means, width = q.double(), means.double(), table.shape[1]
    out = torch.full((T, N, blocks), -1, dtype=torch.int32)
    row = 0
    for b, (count, length) in enumerate(zip(new, lengths)):
        for i in range(count):
            own = (length - count + i) // page
            if length - count + i >= 0 and own < width:
                for n in range(N):
                    qs = q[row, n * (H // N):(n + 1) * (H // N)].sum(0)
                    free = range(min(first, own + 1), max(min(first, own + 1), own + 1 - last))
                    scores = {}
                    for c in free:
                        x = int(table[b, c])
                        s = float(means[x, n] @ qs) if 0 <= x < pages else float("nan")
                        scores[c] = float("-inf") if s != s else s
                    # (a NaN comes behind -inf as well: it sorts by a flag first)
                    nan = lambda c: not 0 <= int(table[b, c]) < pages or bool(torch.isnan(means[int(table[b, c]), n] @ qs))
                    room = max(0, blocks - (own + 1 - len(free)))
                    best = sorted(free, key=lambda c: (nan(c), -scores[c], c))[:room]
                    takes = sorted(best + [c for c in range(own + 1) if c not in free])
                    out[row, n, :len(takes)] = torch.tensor(takes, dtype=torch.int32)
            row += 1
    return out


def select_dense(q, means, table, lengths, new, page, blocks, first, last):
    """select() for many tokens: a sequence's scores at once."""
    T, H, D = q.shape
    pages, N, _ = means.shape
    width = table.shape[1]
    out = torch.full((T, N, blocks), -1, dtype=torch.int32)
    sums = q.double().view(T, N, H // N, D).sum(2)
    at = torch.arange(width)
    row = 0
    for b, (count, length) in enumerate(zip(new, lengths)):
        bad = (table[b] < 0) | (table[b] >= pages)
        m = means[torch.where(bad, 0, table[b]).long()].double()
        own = torch.div(torch.arange(length - count, length), page, rounding_mode="floor")[:, None]
        inside = (own >= 0) & (own < width)
        lo = own.clamp(max=first - 1) + 1
        hi = torch.maximum(lo, own + 1 - last)
        room = (blocks - (own + 1 - (hi - lo))).clamp(min=0)
        for n in range(N):
            scores = sums[row:row + count, n] @ m[:, n].T
            none = bad | torch.isnan(scores)
            scores = torch.where(none, -torch.inf, scores)
            rank = torch.where((at < lo) | (at >= hi), 2, none.long())
            scores, order = torch.sort(scores, dim=1, descending=True, stable=True)
            rank, again = torch.sort(rank.gather(1, order), dim=1, stable=True)
            order = order.gather(1, again)
            taken = torch.zeros((count, width), dtype=torch.bool).scatter_(1, order, (rank < 2) & (at < room))
            taken |= ((at < lo) | (at >= hi)) & (at <= own)
            columns = torch.where(taken & inside, at, width).sort(1).values[:, :blocks]
            columns = torch.where(columns == width, -1, columns).to(torch.int32)
            out[row:row + count, n, :columns.shape[1]] = columns
        row += count
    return out


def attention(q, cache, new, chosen, scale):
    q = q.double()
    out = torch.zeros_like(q)
    N, width, page = cache.cache["k"].shape[1], cache.table.shape[1], cache.page
    row = 0
    for b, (count, length) in enumerate(zip(new, cache.lengths)):
        k, v = cache.rows("k", b, length), cache.rows("v", b, length)
        for i in range(count):
            p = length - count + i
            for h in range(q.shape[1]):
                n = h // (q.shape[1] // N)
                s = [c * page + r for c in chosen[row, n].tolist() if 0 <= c < width for r in range(page) if c * page + r <= p]
                if s:
                    w = torch.softmax(k[s, n] @ q[row, h] * scale, 0)
                    out[row, h] = w @ v[s, n]
            row += 1
    return out


def attention_dense(q, cache, new, chosen, scale):
    """attention() for many tokens: the softmax over all keys, each as often as the token's list shows it."""
    T, H, D = q.shape
    N, width, page = cache.cache["k"].shape[1], cache.table.shape[1], cache.page
    G = H // N
    out = torch.zeros((T, H, D), dtype=torch.float64)
    ends = torch.tensor(new).cumsum(0).tolist()
    for count, end, length, b in zip(new, ends, cache.lengths, range(len(new))):
        if not count or not length:
            continue
        k, v = cache.rows("k", b, length), cache.rows("v", b, length)
        at = torch.arange(length)
        seen = at <= torch.arange(length - count, length)[:, None]
        for n in range(N):
            lists = chosen[end - count:end, n].long()
            lists = torch.where((lists >= 0) & (lists < width), lists, width)
            times = torch.zeros((count, width + 1), dtype=torch.float64).scatter_add_(1, lists, torch.ones(lists.shape, dtype=torch.float64))
            times = times[:, at // page] * seen
            s = q[end - count:end, n * G:(n + 1) * G].double() @ k[:, n].T * scale  # (count, G, length)
            s = torch.where(times[:, None] > 0, s, -torch.inf)
            top = s.amax(-1, keepdim=True).clamp(min=-1e300)
            w = times[:, None] * torch.exp(s - top)
            total = w.sum(-1, keepdim=True)
            out[end - count:end, n * G:(n + 1) * G] = (w / torch.where(total > 0, total, 1.0)) @ v[:, n]
    return out
