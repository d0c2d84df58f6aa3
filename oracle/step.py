"""Oracle: block tables from lengths, verification of drafted tokens and latent
attention, in whole numbers and fp64 numpy from their definitions.

Test infrastructure only (see ``oracle/__init__.py``).  The reference has no
counterpart; the pins (tests/test_oracle_step.py) are closed cases and counted
frequencies.
"""

from __future__ import annotations

import numpy as np

PAGE = 64


def plan_pages(table, held, ctx, new, ring, cursor, length=None, tokens=None):
    """(table, positions, slots, held, cursor, starts), page by page."""
    table, held = np.array(table), [min(max(int(h), 0), np.shape(table)[1]) for h in held]
    taken, returned = int(cursor[0]), int(cursor[1])
    W, F = table.shape[1], len(ring)
    for b in range(len(held)):
        need = -(-(max(int(ctx[b]), 0) + max(int(new[b]), 0)) // PAGE)
        while held[b] < min(need, W) and taken < returned:
            table[b, held[b]] = ring[taken % F]
            held[b] += 1
            taken += 1
    rows, starts = [], [0]
    for b in range(len(held)):
        c, n = max(int(ctx[b]), 0), max(int(new[b]), 0)
        at = [c + t for t in range(n)]
        slot = [int(table[b, p // PAGE]) * PAGE + p % PAGE if p // PAGE < held[b] and table[b, p // PAGE] >= 0 else -1
                for p in at]
        rows.append((at, slot))
        starts.append(starts[-1] + n)
    if length is not None:
        pad = lambda x: (x + [-1] * length)[:length]  # noqa: E731
        pos, slots = ([pad(r[k]) for r in rows] for k in (0, 1))
        starts = []
        pos, slots = (np.array(x, dtype=np.int64).reshape(len(held), length) for x in (pos, slots))
    else:
        pos, slots = ([x for r in rows for x in r[k]] for k in (0, 1))
        pos, slots = (np.array((x + [-1] * tokens)[:tokens], dtype=np.int64) for x in (pos, slots))
    return table, pos, slots, np.array(held, dtype=np.int64), (taken, returned), np.array(starts, dtype=np.int64)


def release_pages(table, held, lens, ring, cursor):
    """(ring, held, cursor)."""
    ring, taken, returned = np.array(ring), int(cursor[0]), int(cursor[1])
    kept = []
    for b, h in enumerate(held):
        h = min(max(int(h), 0), np.shape(table)[1])
        keep = min(h, -(-max(int(lens[b]), 0) // PAGE))
        for i in range(keep, h):
            ring[returned % len(ring)] = table[b][i]
            returned += 1
        kept.append(keep)
    return ring, np.array(kept, dtype=np.int64), (taken, returned)


def _weight(x):
    x = np.asarray(x, dtype=np.float64)
    return np.where(np.isfinite(x) & (x > 0), x, 0.0)


def verify(tokens, target, uniforms, draft=None, parents=None, n=None):
    """One sequence: tokens [T], target [T + 1, V], uniforms [T + 1] -> (kept
    indices, the drawn token or -1)."""
    T, V = len(tokens), target.shape[1]
    n = T if n is None else min(max(int(n), 0), T)
    path, last, refused, left = [], -1, [], 1.0
    p = _weight(target)
    q = _weight(draft) if draft is not None else None
    for i in range(n):
        parent = i - 1 if parents is None else int(parents[i])
        if not -1 <= parent < i or parent != last:
            continue
        x = int(tokens[i])
        px = p[last + 1, x] if 0 <= x < V and x not in [int(tokens[k]) for k in refused] else 0.0
        limit = left if q is None else q[i, x] if 0 <= x < V else 0.0
        if float(uniforms[i]) * limit < px:
            path.append(i)
            last, refused, left = i, [], 1.0
        else:
            refused.append(i)
            left -= px
    row = p[last + 1]
    w = row.copy()
    if refused and q is not None:
        w = np.maximum(row - q[refused[0]], 0.0)
    elif refused:
        w[[int(tokens[k]) for k in refused if 0 <= int(tokens[k]) < V]] = 0.0
    if w.sum() <= 0:
        w = row
    if w.sum() <= 0:
        return path, -1
    u = float(uniforms[T])
    sums = np.cumsum(w)
    above = np.flatnonzero((w > 0) & (sums > max(u, 0.0) * sums[-1]))
    return path, int(above[0]) if above.size else int(np.flatnonzero(w)[-1])


def attend(q, k, v, keep, scale):
    """q [R, E], k [n, E], v [n, D], keep [R, n] -> out, lse, sum of weights x |v|,
    and the largest scale sum |q| |k| of a row's kept keys (what the rounding of
    scores is relative to).  A key that a row does not keep does not reach it; rows
    that keep none are zeros."""
    q, k, v = (np.asarray(x, dtype=np.float64) for x in (q, k, v))
    out, size = np.zeros((len(q), v.shape[1])), np.zeros((len(q), v.shape[1]))
    lse, reach = np.full(len(q), -np.inf), np.zeros(len(q))
    for r in range(len(q)):
        at = np.flatnonzero(keep[r])
        if not at.size:
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            s = scale * (k[at] @ q[r])
            top = s.max()
            e = np.exp(s - top)
            out[r], size[r] = (e / e.sum()) @ v[at], (e / e.sum()) @ np.abs(v[at])
            lse[r] = top + np.log(e.sum())
            reach[r] = abs(scale) * (np.abs(k[at]) @ np.abs(q[r])).max()
    return out, lse, size, reach
