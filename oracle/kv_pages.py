"""Oracle: the pages of a paged cache -- shared, taken, given back -- and accepted rows moved together, a step at a time.

Test infrastructure only (the tests compare the GPU results against it).  A pool is (table [S, W], room [S], ref
[blocks]) as numpy integers, updated in place; ``caches`` are arrays [layers, blocks, page, ...] whose rows move along.
"""
from __future__ import annotations

import numpy as np


def held(room, page):
    return -(-int(room) // page)


def fork(table, room, ref, src, dst, page):
    """Pairs in order; -> whether one was refused.  (Sources are no destinations, so the order does not matter.)"""
    S, W = table.shape
    bad = False
    for i, (a, b) in enumerate(zip(src, dst)):
        if b == -1:
            continue
        clash = any(j != i and (dst[j] == b or (a >= 0 and dst[j] == a)) for j in range(len(dst)))
        if clash or not 0 <= b < S or not -1 <= a < S or not 0 <= room[b] <= W * page or (a >= 0 and not 0 <= room[a] <= W * page):
            bad = True
            continue
        if a == b:
            continue
        had, want = held(room[b], page), held(room[a], page) if a >= 0 else 0
        for j in range(had):
            ref[table[b, j]] -= 1
        for j in range(max(had, want)):
            table[b, j] = table[a, j] if j < want else -1
        for j in range(want):
            ref[table[b, j]] += 1
        room[b] = room[a] if a >= 0 else 0
    return bad


def resize(table, room, ref, new_room, page, caches=()):
    """-> whether a sequence was refused."""
    S, W = table.shape
    bad, out = False, False
    ok = [0 <= n <= W * page and 0 <= r <= W * page for r, n in zip(room, new_room)]
    bad = any(not o and n >= 0 for o, n in zip(ok, new_room))
    for s in range(S):
        if ok[s]:
            for j in range(held(new_room[s], page), held(room[s], page)):
                ref[table[s, j]] -= 1
                table[s, j] = -1
    shared = [ok[s] and new_room[s] > room[s] and room[s] % page > 0 and ref[table[s, held(room[s], page) - 1]] > 1 for s in range(S)]
    for s in range(S):
        if not ok[s]:
            continue
        want = held(new_room[s], page)
        kept = min(held(room[s], page), want)
        copy = shared[s] and ref[table[s, kept - 1]] > 1
        free = np.flatnonzero(ref == 0)
        need = want - kept + copy
        if (need or shared[s]) and (out or need > len(free)):
            bad = out = True
            continue
        if copy:
            old, n = int(table[s, kept - 1]), int(room[s]) % page
            for c in caches:
                c[:, free[0], :n] = c[:, old, :n]
            ref[old] -= 1
            kept -= 1
        table[s, kept:want] = free[:need]
        ref[free[:need]] += 1
        room[s] = new_room[s]
    return bad


def commit(caches, table, lens, path, count, page):
    """Rows moved one after the other; -> whether a sequence was refused."""
    blocks, W = caches[0].shape[1], table.shape[1]
    bad = False

    def slot(s, pos):
        b = int(table[s, pos // page]) if pos < W * page else -1
        return (b, pos % page) if 0 <= b < blocks else None
    for s, n in enumerate(count):
        if n < 1:
            continue
        p = [int(v) for v in path[s][:n]]
        if n > path.shape[1] or lens[s] < 0 or any(b <= a for a, b in zip([-1] + p, p)) or any(
                slot(s, int(lens[s]) + v) is None for v in p + list(range(n))):
            bad = True
            continue
        for i, v in enumerate(p):
            a, b = slot(s, int(lens[s]) + v), slot(s, int(lens[s]) + i)
            for c in caches:
                c[:, b[0], b[1]] = c[:, a[0], a[1]]
    return bad


def check(table, room, ref, page):
    """The invariants of a pool that only these calls have changed: every sequence holds as many pages as its room takes
    and none behind, every page is counted by its holders, and no sequence holds a page twice."""
    count = np.zeros_like(ref)
    for s in range(len(table)):
        n = held(room[s], page)
        row = table[s, :n]
        assert (row >= 0).all() and (table[s, n:] == -1).all() and len(set(row.tolist())) == n
        count[row] += 1
    assert np.array_equal(count, ref)
