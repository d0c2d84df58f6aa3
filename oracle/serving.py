"""Oracle: rotary positions, the 8-bit paged cache and attention of drafted
tokens, in fp64 numpy from their definitions.

Test infrastructure only (see ``oracle/__init__.py``).  The reference has no
counterpart; the pins (tests/test_oracle_serving.py) are closed cases: a turn
of a quarter, norms kept, the type's own numbers stored exactly, ties to even,
one attended token, the chain mask against causal SDPA.
"""

from __future__ import annotations

import math

import numpy as np

PAGE = 64
TOP = {"e4m3": 448.0, "int8": 127.0}


def rotate(x, positions, frequencies, amplitude=1.0, interleaved=False, inverse=False):
    """x [..., S, D] with pair i of row s turned by positions[..., s] *
    frequencies[i] (positions broadcast against x's leading dimensions)."""
    x = np.asarray(x, dtype=np.float64)
    f = np.asarray(frequencies, dtype=np.float64)
    n = f.size
    theta = np.asarray(positions).astype(np.float64)[..., None] * f
    c, s = amplitude * np.cos(theta), amplitude * np.sin(theta)
    if inverse:
        s = -s
    y = x.copy()
    i1, i2 = (np.arange(0, 2 * n, 2), np.arange(1, 2 * n, 2)) if interleaved else (np.arange(n), np.arange(n, 2 * n))
    y[..., i1] = x[..., i1] * c - x[..., i2] * s
    y[..., i2] = x[..., i2] * c + x[..., i1] * s
    return y


def e4m3_nearest(y):
    """The nearest e4m3 number (3 mantissa bits, exponents from -6), ties to even."""
    y = np.asarray(y, dtype=np.float64)
    _, e = np.frexp(y)
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)
    return np.rint(y / step) * step


def quantise(x, codes):
    """Rows x [..., D] -> (the numbers that the codes are, scale [...])."""
    x = np.asarray(x, dtype=np.float64)
    top = np.abs(x).max(axis=-1)
    top = np.where(top >= 2.0 ** -100, top, TOP[codes])
    y = x * TOP[codes] / top[..., None]
    return (np.rint(y) if codes == "int8" else e4m3_nearest(y)), (top / TOP[codes]).astype(np.float32)


def pages8_to_logical(k, v):
    """Codes (as numbers) in page layout -> [P, H, 64, D] each."""
    P, H, U, T, _ = k.shape
    return (k.transpose(0, 1, 3, 2, 4).reshape(P, H, T, U * 16),
            v.transpose(0, 1, 2, 4, 3).reshape(P, H, T, v.shape[3]))


def gather(pages, row, n):
    """The first n tokens [H, n, ...] of logical pages [P, H, 64, ...]."""
    idx = np.asarray(row[:max(1, -(-n // PAGE))], dtype=np.int64)
    x = np.moveaxis(pages[idx], 1, 0)
    return x.reshape((x.shape[0], -1) + x.shape[3:])[:, :n]


def tree_keep(ctx, n, T, mask=None):
    """keep [T, ctx + n]: what each query row attends; rows from n on nothing."""
    keep = np.zeros((T, ctx + n), dtype=bool)
    m = np.tril(np.ones((T, T), dtype=bool)) if mask is None else np.asarray(mask, dtype=bool)
    keep[:n, :ctx] = True
    keep[:n, ctx:] = m[:n, :n]
    return keep


def attend(q, k, v, keep, scale=None):
    """q [T, Hq, D], k / v [Hkv, n, D], keep [T, n] -> out [T, Hq, D], lse [T,
    Hq] and the weighted mean of |v| that bounds the rounding of the weights.
    A key that a row does not keep does not reach it, whatever it holds."""
    q, k, v = (np.asarray(x, dtype=np.float64) for x in (q, k, v))
    T, Hq, D = q.shape
    g = Hq // k.shape[0]
    s = 1.0 / math.sqrt(D) if scale is None else scale
    out, size = np.zeros((T, Hq, D)), np.zeros((T, Hq, D))
    lse = np.full((T, Hq), -np.inf)
    for i in range(T):
        at = np.flatnonzero(keep[i])
        if not at.size:
            continue
        for h in range(Hq):
            with np.errstate(invalid="ignore"):
                score = s * (k[h // g][at] @ q[i, h])
                top = score.max()
                e = np.exp(score - top)
                out[i, h] = (e / e.sum()) @ v[h // g][at]
                size[i, h] = (e / e.sum()) @ np.abs(v[h // g][at])
                lse[i, h] = top + np.log(e.sum())
    return out, lse, size
