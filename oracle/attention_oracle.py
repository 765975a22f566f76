"""The attention operators in 64 bits, written from their definitions (numpy, one sequence and head at a time).

No counterpart in the reference's projection path: these are this package's
own operators, and the definitions stand in ``include/langburst_lowbit.h``.
"""
from __future__ import annotations

import numpy as np


def rotate(x, cos, sin, interleaved):
    """x [..., head_dim] with the angles of its position: the first 2 * len(cos) values turn, pairs (a, b) -> (a cos - b sin, b cos + a sin)."""
    out = np.array(x, dtype=np.float64)
    n = len(cos)
    a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    u, w = out[..., a].copy(), out[..., b].copy()
    out[..., a], out[..., b] = u * cos - w * sin, w * cos + u * sin
    return out


def attend(q, k, v, scale, sees):
    """q [n, d] over k, v [m, d]; row i sees the keys 0 .. sees[i] - 1; a row that sees none is zero.

    Returns (output, sum_j p_j |v_j|, sum_j |v_j|): the last two bound the error
    of rounded weights."""
    q, k, v = (np.asarray(t, dtype=np.float64) for t in (q, k, v))
    out, spread, total = np.zeros((len(q), v.shape[1])), np.zeros((len(q), v.shape[1])), np.zeros((len(q), v.shape[1]))
    for i, m in enumerate(sees):
        m = min(max(int(m), 0), len(k))
        if m == 0:
            continue
        s = (k[:m] @ q[i]) * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        out[i], spread[i], total[i] = p @ v[:m], p @ np.abs(v[:m]), np.abs(v[:m]).sum(0)
    return out, spread, total


def score_error(q, k, scale):
    """Bound of the error of a score summed in fp32 (any order): (d + 3) 2^-24 sum |q k| scale, over all rows and keys."""
    q, k = np.abs(np.asarray(q, dtype=np.float64)), np.abs(np.asarray(k, dtype=np.float64))
    if not len(q) or not len(k):
        return 0.0
    return (q.shape[1] + 3) * 2.0 ** -24 * float((q @ k.T).max()) * scale
