"""The fixed-point model operators from their definitions, in 64-bit integers on the host."""
import math

import numpy as np


def rs(a, shift):
    return np.floor_divide(a + ((1 << shift) >> 1), 1 << shift)


def sat(a):
    return np.clip(a, -32768, 32767)


def linear(x, w, *, bias=None, bias_shift=0, shift=0, table=None, residual=None, raw=False):
    acc = x.astype(np.int64) @ w.astype(np.int64)
    if bias is not None:
        acc = acc + bias.astype(np.int64) * (1 << bias_shift)
    if raw:
        return acc
    h = sat(rs(acc, shift))
    if table is not None:
        h = table.astype(np.int64)[h + 32768]
    if residual is not None:
        h = sat(h + residual.astype(np.int64))
    return h.astype(np.int16)


def _sums(a, b):
    """a @ b of integers below 2^15 and 2^16 in size, over fewer than 2^21 terms: exact in doubles."""
    return (a.astype(np.float64) @ b.astype(np.float64)).astype(np.int64)


def attention(q, keys, values, table, shift, causal):
    """q: rows x heads x dim; keys, values: tokens x kv heads x dim; the rows are the last tokens."""
    rows, heads, _ = q.shape
    tokens, kv_heads, _ = keys.shape
    out = np.zeros(q.shape, np.int16)
    if tokens == 0:
        return out
    e_of = np.minimum(table.astype(np.int64), 1 << 14)
    hidden = np.zeros((rows, tokens), bool)
    if causal:
        hidden = np.arange(tokens)[None, :] > (tokens - rows + np.arange(rows))[:, None]
    for h in range(heads):
        k, v = (t[:, h * kv_heads // heads] for t in (keys, values))
        z = _sums(q[:, h], k.T) >> shift
        z[hidden] = -(1 << 60)
        e = e_of[np.minimum(z.max(1, keepdims=True) - z, len(e_of) - 1)]
        e[hidden] = 0
        total = e.sum(1, keepdims=True)
        out[:, h] = np.where(total > 0, np.floor_divide(2 * _sums(e, v) + total, np.maximum(2 * total, 1)), 0)
    return out


def norm(x, gain, shift, eps, *, bias=None, residual=None, rms=False):
    """(y, h)"""
    h = x.astype(np.int64)
    if residual is not None:
        h = sat(h + residual.astype(np.int64))
    n = x.shape[1]
    y = np.empty(h.shape, np.int64)
    for i, row in enumerate(h):
        s = 0 if rms else int(row.sum())
        below = math.isqrt(n * int((row * row).sum()) - s * s + eps) << shift
        y[i] = np.floor_divide(2 * (n * row - s) * gain.astype(np.int64) + below, 2 * below)
    if bias is not None:
        y = y + bias.astype(np.int64)
    return sat(y).astype(np.int16), h.astype(np.int16)


def embed(tokens, table, *, scale=1, shift=0, positions=None, position_table=None):
    out = np.zeros((len(tokens), table.shape[1]), np.int64)
    for i, t in enumerate(tokens):
        if 0 <= t < len(table):
            out[i] = rs(table[t].astype(np.int64) * scale, shift)
        if positions is not None and 0 <= positions[i] < len(position_table):
            out[i] += position_table[positions[i]]
    return sat(out).astype(np.int16)
