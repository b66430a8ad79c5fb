"""The paged cache's allocator from its definition, one row and page after the other: the oracle of its
kernels' tests."""

from __future__ import annotations

import random


def ceil(a, b):
    return -(-a // b)


def used_entries(row, length, page):
    return row[:min(len(row), ceil(max(0, length), page))]


def extend(table, lengths, parents, new, pages, page):
    """(table, lengths, free pages, [(from, to, rows)]) after rows went on from parents and grew by new."""
    batch, width = len(table), len(table[0])
    rows, held = [], []
    for b in range(batch):
        p = b if parents is None else parents[b]
        there = 0 <= p < batch
        held.append(max(0, lengths[p]) if there else 0)
        rows.append(used_entries(list(table[p]), held[b], page) if there else [])
    grows = [new[b] > 0 and held[b] % page != 0 and ceil(held[b], page) <= width for b in range(batch)]
    users = {}  # page: rows that go on reading it as it is count as -1
    for b, row in enumerate(rows):
        for c, x in enumerate(row):
            if 0 <= x < pages:
                users.setdefault(x, []).append(b if grows[b] and c == len(row) - 1 else -1)
    free = [x for x in range(pages) if x not in users]
    left, at, copies = len(free), 0, []
    for b, row in enumerate(rows):
        last = row[-1] if row else -1
        copy = grows[b] and 0 <= last < pages and min(users[last]) != b
        want = max(0, min(width, ceil(held[b] + max(0, new[b]), page)) - len(row)) + copy
        got = [free[i] if i < len(free) else -1 for i in range(at, at + want)]
        at += want
        left -= want
        if copy:
            if got[0] >= 0:
                copies.append((last, got[0], held[b] % page))
            row.pop()
        rows[b] = row + got
    table = [row + [-1] * (width - len(row)) for row in rows]
    return table, [min(h + max(0, n), 2 ** 31 - 1) for h, n in zip(held, new)], left, copies


def compact(table, lengths, pages, page, out_pages):
    """(the used pages in order, the new table)."""
    used = sorted({x for row, n in zip(table, lengths) for x in used_entries(row, n, page) if 0 <= x < pages})
    place = {x: i for i, x in enumerate(used) if i < out_pages}
    table = [[place.get(x, -1) if c < len(used_entries(row, n, page)) else -1 for c, x in enumerate(row)]
             for row, n in zip(table, lengths)]
    return used, table


def scenario(seed, batch, width, pages, page, wild=True):
    """Rows that share pages, fully and in their last ones, at equal and unequal lengths; wild: also entries
    outside the cache, lengths below zero and beyond the table, parents outside the batch, a page twice in a row."""
    rng = random.Random(seed)
    ids = list(range(pages))
    rng.shuffle(ids)
    table, lengths = [], []
    for b in range(batch):
        length = rng.choice((0, 1, page - 1, page, page + 1, rng.randint(0, width * page), rng.randint(0, width * page)))
        if table and rng.random() < 0.5:  # a fork of an earlier row, shorter, as long or longer
            other = rng.randrange(len(table))
            row = list(table[other])
            length = rng.choice((lengths[other], max(0, lengths[other] - rng.randint(0, 2 * page)), length))
        else:
            row = [-1] * width
        for c in range(min(width, ceil(max(0, length), page))):
            if row[c] == -1:
                row[c] = ids.pop() if ids else rng.randrange(pages)
        if wild and rng.random() < 0.2:
            row[rng.randrange(width)] = rng.choice((-5, pages, 2 ** 31 - 1, row[0]))
        if wild and rng.random() < 0.1:
            length = rng.choice((-3, width * page + 5, 2 ** 31 - 4))
        table.append(row)
        lengths.append(length)
    parents = None if rng.random() < 0.3 else [
        rng.choice((b, rng.randrange(batch), rng.randrange(batch), -1 if wild else b, batch if wild else b))
        for b in range(batch)]
    new = [rng.choice((0, 1, 1, 1, page, rng.randint(0, 3 * page), -4 if wild else 2)) for _ in range(batch)]
    return table, lengths, parents, new
