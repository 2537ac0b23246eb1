"""The serving operators from their definitions, in whole numbers on the host: heads normed and rotated, attention over
a window or behind a prefix, and the choice of the next token."""
import math

import fixed_reference as ref
import numpy as np


def attention(q, keys, values, seen, table, shift):
    """q: rows x heads x dim; keys, values: tokens x kv heads x dim; seen: rows x tokens."""
    rows, heads, _ = q.shape
    tokens, kv_heads, _ = keys.shape
    out = np.zeros(q.shape, np.int16)
    if tokens == 0 or rows == 0:
        return out
    e_of = np.minimum(table.astype(np.int64), 1 << 14)
    for h in range(heads):
        k, v = (t[:, h * kv_heads // heads] for t in (keys, values))
        z = ref._sums(q[:, h], k.T) >> shift
        z[~seen] = -(1 << 60)
        e = e_of[np.minimum(z.max(1, keepdims=True) - z, len(e_of) - 1)]
        e[~seen] = 0
        total = e.sum(1, keepdims=True)
        out[:, h] = np.where(total > 0, np.floor_divide(2 * ref._sums(e, v) + total, np.maximum(2 * total, 1)), 0)
    return out


def window_seen(rows, tokens, window, sinks):
    """Which of `tokens` keys the last `rows` of them see."""
    j, p = np.arange(tokens)[None, :], (tokens - rows + np.arange(rows))[:, None]
    return (j <= p) & ((j > p - window) | (j < sinks))


def prefix_seen(rows, prefix, tokens, causal):
    """Which keys of a prefix and a sequence behind it the sequence's last `rows` see."""
    seen = np.ones((rows, prefix + tokens), bool)
    if causal:
        seen[:, prefix:] = np.arange(tokens)[None, :] <= (tokens - rows + np.arange(rows))[:, None]
    return seen


def rotate(x, heads, dim, *, q_gain=None, k_gain=None, gain_shift=0, eps=1, angles=None, positions=None, rotated=0,
           adjacent=False, angle_shift=14):
    """x: rows x (heads of queries and keys * dim)"""
    h = x.astype(np.int64).reshape(len(x), -1, dim)
    for at, gain in ((slice(0, heads), q_gain), (slice(heads, None), k_gain)):
        if gain is None:
            continue
        for row in (r for token in h[:, at] for r in token):
            below = math.isqrt(dim * int((row * row).sum()) + eps) << gain_shift
            row[:] = ref.sat(np.floor_divide(2 * dim * row * gain.astype(np.int64) + below, 2 * below))
    out = h.copy()
    for row, place in enumerate(positions if rotated else ()):
        if not 0 <= place < len(angles):
            continue
        for i in range(rotated // 2):
            one, two = (2 * i, 2 * i + 1) if adjacent else (i, i + rotated // 2)
            c, s = (int(v) for v in angles[place, i])
            a, b = h[row, :, one], h[row, :, two]
            out[row, :, one] = ref.sat(ref.rs(a * c - b * s, angle_shift))
            out[row, :, two] = ref.sat(ref.rs(a * s + b * c, angle_shift))
    return out.reshape(x.shape).astype(np.int16)


def choose(logits, rows, *, bias_shift=0):
    """(tokens, adjusted) with a dict of history, biases, mask, frequency, presence and repetition for each row."""
    out, tokens = np.empty(logits.shape, np.int64), np.empty(len(logits), np.int32)
    vocab = logits.shape[1]
    most = (1 << 63) - 1
    for i, r in enumerate(rows):
        l = [int(v) for v in logits[i]]
        counts, biases = {}, {}
        for t in r["history"]:
            counts[int(t)] = counts.get(int(t), 0) + 1
        for t, v in r["biases"]:
            biases[int(t)] = biases.get(int(t), 0) + int(v)
        for t, n in counts.items():
            if 0 <= t < vocab:
                rep = r["repetition"]
                x = (l[t] * rep + (1 << 15)) >> 16 if l[t] < 0 else (2 * (l[t] << 16) + rep) // (2 * rep)
                l[t] = x - r["frequency"] * n - r["presence"]
        for t, v in biases.items():
            if 0 <= t < vocab:
                l[t] += v << bias_shift
        l = [max(-most, min(most, v)) for v in l]
        if r["mask"] is not None:
            l = [v if ok else -most - 1 for v, ok in zip(l, r["mask"])]
        best = max(l)
        tokens[i] = -1 if best == -most - 1 else l.index(best)
        out[i] = l
    return tokens, out
