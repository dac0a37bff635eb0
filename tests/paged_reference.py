"""Plain 64-bit implementations of the paged-cache operators, for their tests:
wrapping int64 sums in numpy, the softmax of the oracle (det-num in C)."""
import ctypes as C

import numpy as np

from oracle import cpu

I32_MIN, I32_MAX = -(1 << 31), (1 << 31) - 1


def _rte16(x):
    low = x >> 16
    return low + ((x & 0xFFFF) + (low & 1) > 0x8000)


def scores(q, k, scale):
    """[rows][keys] scores of int32 rows and keys (scale 0: unscaled)."""
    with np.errstate(over="ignore"):
        dot = np.stack([(row.astype(np.int64)[None, :] * k.astype(np.int64)).sum(axis=1) for row in q]) \
            if len(q) else np.zeros((0, len(k)), np.int64)
        if scale:
            dot = (dot >> 32) * scale + (((dot & 0xFFFFFFFF).astype(np.uint64) * np.uint64(scale)) >> np.uint64(32)).astype(np.int64)
    return np.clip(_rte16(dot), I32_MIN, I32_MAX).astype(np.int32)


def attend(q, k, v, seen, scale):
    """One head: rows [n][hd] over keys [m][hd] where seen [n][m]."""
    L = cpu.lib()
    sc = scores(q, k, scale)
    out = np.zeros_like(q)
    for i in range(len(q)):
        keys = np.flatnonzero(seen[i])
        logits = np.ascontiguousarray(sc[i, keys])
        w = np.empty(len(keys), np.int32)
        L.dn_attention_softmax(logits, len(keys), np.empty(len(keys), np.int64), w)
        with np.errstate(over="ignore"):
            total = (w.astype(np.int64)[:, None] * v[keys].astype(np.int64)).sum(axis=0)
        out[i] = np.clip(_rte16(total), I32_MIN, I32_MAX)
    return out


def packed(q, k, v, starts, heads, kv_heads, hd, window, scale, out):
    """Rows of packed sequences into out (rows past the last left)."""
    for a, b in zip(starts[:-1], starts[1:]):
        n = b - a
        at = np.arange(n)
        seen = (at[None, :] <= at[:, None]) & ((at[:, None] - at[None, :] < window) if window else True)
        for h in range(heads):
            g = h // (heads // kv_heads)
            qs, ks = slice(h * hd, h * hd + hd), slice(g * hd, g * hd + hd)
            out[a:b, qs] = attend(q[a:b, qs], k[a:b, ks], v[a:b, ks], seen, scale)
    return out


def ancestors(parents):
    """Each row's set of rows up its tree, itself included."""
    above = []
    for i, p in enumerate(parents):
        above.append((above[p] if 0 <= p < i else set()) | {i})
    return above


def tree_mask(length, parents, window):
    """seen [rows][length + rows] and the rows' positions."""
    above = ancestors(parents)
    n = len(parents)
    pos = [length + len(a) - 1 for a in above]
    seen = np.zeros((n, length + n), bool)
    for i in range(n):
        seen[i, max(0, pos[i] + 1 - window) if window else 0:length] = True
        for j in above[i]:
            seen[i, length + j] = not window or pos[i] - pos[j] < window
    return seen, pos


def tree(q, k_pages, v_pages, table, starts, lengths, parents, heads, window, scale, out):
    """Drafted rows over pages [pages][kv_heads][page_size][hd]; a page
    outside the cache reads as zeros."""
    pages, kv_heads, page, hd = k_pages.shape
    for i, (a, b) in enumerate(zip(starts[:-1], starts[1:])):
        n, m = b - a, lengths[i] + b - a
        if n <= 0:
            continue
        par = list(range(-1, n - 1)) if parents is None else list(parents[a:b])
        seen, _ = tree_mask(lengths[i], par, window)
        at = np.arange(m)
        ids = table[i][at // page].astype(np.int64)
        good = (ids >= 0) & (ids < pages)
        ids = np.where(good, ids, 0)
        for h in range(heads):
            g = h // (heads // kv_heads)
            k = k_pages[ids, g, at % page] * good[:, None]
            v = v_pages[ids, g, at % page] * good[:, None]
            cols = slice(h * hd, h * hd + hd)
            out[a:b, cols] = attend(q[a:b, cols], k.astype(np.int32), v.astype(np.int32), seen, scale)
    return out


def plan(lengths, added, parents, held, table, ring, ring_state, pages, page, max_rows):
    """(table, held, ring, ring_state, row_start, slots, positions, status)."""
    n, stride = table.shape
    held, table, ring = list(held), table.copy(), list(ring)
    head, free = ring_state
    fail = [table, np.array(held), np.array(ring), np.array(ring_state), np.zeros(n + 1, int), np.full(max_rows, -1),
            np.full(max_rows, -1)]
    need = [-(-(x + a) // page) for x, a in zip(lengths, added)]
    if not (0 <= head < pages and 0 <= free <= pages) or any(
            x < 0 or a < 0 or h < 0 or h > stride or h * page < x for x, a, h in zip(lengths, added, held)):
        return *fail, -1
    grow = sum(max(0, d - h) for d, h in zip(need, held))
    back = sum(max(0, h - d) for d, h in zip(need, held))
    if max(need) > stride or sum(added) > max_rows or grow > free or (parents is not None and max(added) > 64):
        return *fail, -5
    if free + back > pages:
        return *fail, -1
    slots, positions, starts, taken, given = [], [], [0], 0, []
    for i in range(n):
        for j in range(held[i], need[i]):
            table[i, j] = ring[(head + taken) % pages]
            taken += 1
        given += [table[i, j] for j in range(need[i], held[i])]
        par = range(-1, added[i] - 1) if parents is None else parents[starts[-1]:starts[-1] + added[i]]
        above = ancestors(list(par)) if parents is not None else None
        for r in range(added[i]):
            at = lengths[i] + r
            p = table[i, at // page]
            slots.append(p * page + at % page if 0 <= p < pages else -1)
            positions.append(at if above is None else lengths[i] + len(above[r]) - 1)
        starts.append(starts[-1] + added[i])
    for j, p in enumerate(given):
        ring[(head + free + j) % pages] = p
    tail = [-1] * (max_rows - len(slots))
    return (table, np.array(need), np.array(ring), np.array([(head + taken) % pages, free - taken + back]),
            np.array(starts), np.array(slots + tail), np.array(positions + tail), 0)
