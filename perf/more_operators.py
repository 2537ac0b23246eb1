"""Timed cases of the operators that serve the committed model: rotated and normed heads, attention over a window or
a shared prefix, and the choice of the next token.

Everything is an integer with an exact definition, so every correct
implementation gives the same values.  rs(a, s) is a / 2^s rounded to the
nearest integer, halves up (a for s = 0); sat clamps to 16 bits.

rotate  heads of queries and keys in one pass.  With a gain: n = dim, V = n sum h^2 + eps,
        R = floor(sqrt(V)), h = sat(n h gain / (R 2^gain_shift), rounded to nearest, halves up).
        Then, for i < rotated / 2 with (c, s) = angles[position][i] at 2^-14, the places
        (i, i + rotated / 2), or (2 i, 2 i + 1) if adjacent: a' = sat(rs(a c - b s, 14)),
        b' = sat(rs(a s + b c, 14)).  Other places stay.
window  z = (q . k) >> shift, e = table[min(max z - z, len - 1)], out = sum e v / sum e rounded
        to nearest, halves up, over the keys at places j <= p, the row's own, with j > p - window or j < sinks.
shared  the same over the tokens of a prefix that all sequences share, then the sequence's own up to the row's.
choose  of a row's logits: a token that occurs n > 0 times in its history gets l r / 2^16 (l < 0)
        or l 2^16 / r (l >= 0), both rounded to nearest, halves up, less frequency n + presence;
        then its biases are added, and tokens that are not allowed get -2^63.  Results: the lowest
        index of the largest allowed logit (-1: none), and the logits where asked for.

The plain forms work in 64 bits: products of 16-bit values summed over a head
pass 2^24, and so do the logits.
"""
from __future__ import annotations

import math
import pathlib
import random
import sys

import numpy as np
import torch

own = False

ENTRIES = 8192  # of the exponential table
MOST_ELEMENTS = 16384 * 24 * 64  # of the largest listed rotate case
MOST_WINDOW_PAIRS = 16 * 16384 * 1024  # head x query x visible key places of the largest listed window case
MOST_SHARED_PAIRS = 1 << 26  # under the largest listed shared case's
MOST_LOGITS = 256 * 50257
QUERIES = 512  # rows that the plain form of the window takes at a time


# ---- the cases ------------------------------------------------------------------------------

def listed() -> list[dict]:
    return [
        # One generated token's queries and keys, 12 heads of 64: latency.
        dict(name="rotate_token", kind="rotate", rows=1, heads=12, kv_heads=12, dim=64, rotated=64, adjacent=False,
             gains=True, positions=1024, gap=768),
        # A long prompt with grouped heads of 128, three quarters of each rotated, without norms.
        dict(name="rotate_partial", kind="rotate", rows=4095, heads=32, kv_heads=8, dim=128, rotated=96, adjacent=True,
             gains=False, positions=8192, gap=13),
        # Sixteen contexts in the layout of a joint product for queries, keys and values.
        dict(name="rotate_batch", kind="rotate", rows=16384, heads=12, kv_heads=12, dim=64, rotated=64, adjacent=False,
             gains=True, positions=1024, gap=768),
        # One token of one sequence, far behind its first ones.
        dict(name="window_token", kind="window", batch=1, new=1, longest=4096, ragged=0, heads=12, kv_heads=12, dim=64,
             window=512, sinks=4),
        # One token each of 64 sequences of different lengths, grouped heads.
        dict(name="window_tokens", kind="window", batch=64, new=1, longest=4095, ragged=5, heads=32, kv_heads=8,
             dim=128, window=1024, sinks=16),
        # One long prompt, grouped heads of 128.
        dict(name="window_long", kind="window", batch=1, new=0, longest=16384, ragged=0, heads=16, kv_heads=4, dim=128,
             window=1024, sinks=4),
        # One token each of four sequences behind instructions that they share.
        dict(name="shared_few", kind="shared", batch=4, new=1, prefix=1000, longest=24, ragged=3, heads=12, kv_heads=12,
             dim=64),
        # One token each of 64 sequences behind a long document, grouped heads.
        dict(name="shared_tokens", kind="shared", batch=64, new=1, prefix=8192, longest=255, ragged=7, heads=32,
             kv_heads=8, dim=128),
        # Sixteen questions of different lengths about the same document.
        dict(name="shared_prompts", kind="shared", batch=16, new=0, prefix=2047, longest=400, ragged=9, heads=12,
             kv_heads=12, dim=64),
        # The next token of one sequence, repeated tokens made less likely.
        dict(name="choose_token", kind="choose", rows=1, vocab=50257, history=200, biases=0, masked=False,
             adjusted=False),
        # 64 sequences under a grammar, with biases, the logits kept.
        dict(name="choose_batch", kind="choose", rows=64, vocab=50257, history=1023, biases=50, masked=True,
             adjusted=True),
        # 256 long sequences; only their tokens are wanted.
        dict(name="choose_many", kind="choose", rows=256, vocab=50257, history=8191, biases=300, masked=True,
             adjusted=False),
    ]


def _log(rng, lo: int, hi: int) -> int:
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(2.0 ** rng.uniform(math.log2(lo), math.log2(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["rotate", "window", "window", "shared", "shared", "choose"])
    if kind == "choose":
        vocab, adjusted = _log(rng, 100, 100000), rng.random() < 0.5
        return dict(kind=kind, rows=_log(rng, 1, min(256, MOST_LOGITS // (vocab * (1 + adjusted)))), vocab=vocab,
                    history=_log(rng, 1, 8191), biases=rng.choice([0, 0, 1, 17, 300]), masked=rng.random() < 0.6,
                    adjusted=adjusted)
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    dim = rng.choice([32, 40, 64, 64, 80, 96, 128, 128])
    if kind == "rotate":
        return dict(kind=kind, rows=_log(rng, 1, min(16384, MOST_ELEMENTS // ((heads + kv_heads) * dim))), heads=heads,
                    kv_heads=kv_heads, dim=dim, rotated=rng.choice([dim, dim, dim // 2, 2 * rng.randint(0, dim // 2)]),
                    adjacent=rng.random() < 0.4, gains=rng.random() < 0.7, positions=_log(rng, 16, 16384),
                    gap=rng.choice([0, kv_heads * dim, 8, 13]))
    batch = _log(rng, 1, 64)
    if kind == "window":
        window, sinks = _log(rng, 16, 2048), rng.choice([0, 1, 4, 16, 64, 100])
        if rng.random() < 0.5:  # tokens over a cache
            new = _log(rng, 1, 8)
            longest = max(new, _log(rng, 1, min(16384, (1 << 28) // (batch * kv_heads * dim))))
        else:  # whole prompts
            new, most = 0, MOST_WINDOW_PAIRS // (batch * heads * (window + sinks))
            longest = _log(rng, 1, max(1, min(16384, most, (1 << 28) // (batch * kv_heads * dim))))
            while batch * heads * min(longest, QUERIES) * (min(window, longest) + QUERIES + sinks) > 1 << 28:
                longest //= 2  # the plain form's scores of a block of rows
        return dict(kind=kind, batch=batch, new=new, longest=longest, ragged=rng.randint(0, 1 << 20), heads=heads,
                    kv_heads=kv_heads, dim=dim, window=window, sinks=sinks)
    prefix = _log(rng, 16, 16384)
    new = _log(rng, 1, 4) if rng.random() < 0.6 else 0
    longest = max(new, _log(rng, 1, 512))
    while batch > 1 and batch * heads * (new or longest) * (prefix + longest) > MOST_SHARED_PAIRS:
        batch //= 2
    while new == 0 and longest > 1 and batch * heads * longest * (prefix + longest) > MOST_SHARED_PAIRS:
        longest //= 2
    return dict(kind=kind, batch=batch, new=new, prefix=prefix, longest=longest, ragged=rng.randint(0, 1 << 20),
                heads=heads, kv_heads=kv_heads, dim=dim)


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """(new tokens, tokens in all) of each sequence; ``ragged`` seeds lengths from the longest's fourth part on."""
    longest, batch = case["longest"], case["batch"]
    if case["ragged"]:
        r = random.Random(case["ragged"])
        total = [longest] + [r.randint(max(1, case["new"], longest // 4), longest) for _ in range(batch - 1)]
    else:
        total = [longest] * batch
    return [case["new"] or t for t in total], total


# ---- inputs ---------------------------------------------------------------------------------

class _State:
    """A case's inputs on the GPU."""


class _Region:
    """Device memory of a resident buffer as torch sees it."""

    def __init__(self, ptr: int, shape, typestr: str, keep):
        self.keep = keep
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (ptr, False),
                                         "version": 3, "strides": None}


class _Resident:
    """The same inputs as a user of the library holds them: resident buffers,
    returned to the pool with the state."""

    def __init__(self):
        root = pathlib.Path(__file__).resolve().parents[1] / "volta-zk_amd"
        if str(root) not in sys.path:
            sys.path.insert(0, str(root))
        from volta_mi355x import accel
        global _backend
        if _backend is None:  # the one context that a serving process keeps, counting its calls without events
            _backend = accel.Backend(timing_policy=1)
        self.b, self.bufs, self.kept = _backend, [], []
        if self.b.memory_breakdown()[2] > 64 << 30:
            self.b.lib.volta_cuda_trim_resident_cache(self.b.raw)

    def view(self, buf, shape, typestr):
        return torch.as_tensor(_Region(self.b.device_ptr(buf), shape, typestr, self), device="cuda")

    def new(self, shape, dtype):
        buf = self.b.alloc_device(math.prod(shape), dtype)
        self.bufs.append(buf)
        return buf, self.view(buf, shape, np.dtype(dtype).str)

    def put(self, t: torch.Tensor):
        if t is None:
            return None
        buf, view = self.new(t.shape, {torch.int16: np.int16, torch.int32: np.int32, torch.int64: np.int64}[t.dtype])
        self.b.synchronize()  # torch writes on a stream of its own
        view.copy_(t)
        torch.cuda.synchronize()
        return buf

    def __del__(self):
        for buf in self.bufs:
            self.b.free_device(buf)
        for free, handle in self.kept:
            free(handle)


_backend = None


def _normal(g, shape, std) -> torch.Tensor:
    """Quantised values: i16 ~ N(0, std^2), rounded and clipped."""
    return torch.randn(shape, generator=g, device="cuda").mul_(std).round_().clamp_(-32768, 32767).to(torch.int16)


def _integers(g, lo, hi, shape, dtype=torch.int32) -> torch.Tensor:
    return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=dtype)


def _exponentials() -> torch.Tensor:
    """2^14 exp(-i / 640): 0 in the last entry."""
    i = np.arange(ENTRIES)
    return torch.from_numpy(np.rint(16384.0 * np.exp(-i / 640.0)).astype(np.int16)).cuda()


def _angles(positions: int, pairs: int) -> torch.Tensor:
    """(cos, sin) at 2^-14 of position / 10,000^(i / pairs)."""
    a = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(pairs) / max(1, pairs))
    return torch.from_numpy(np.rint(16384.0 * np.stack([np.cos(a), np.sin(a)], -1)).astype(np.int16)).cuda()


def _inputs(case: dict, seed: int) -> _State:
    """What the case reads, as tensors: ``exact`` and both forms of ``run`` start from these."""
    s, kind = _State(), case["kind"]
    s.case = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if kind == "rotate":
        rows, dim = case["rows"], case["dim"]
        s.x = _normal(g, (rows, (case["heads"] + case["kv_heads"]) * dim + case["gap"]), 1500.0)
        s.q_gain = _normal(g, (dim,), 600.0).add_(4096) if case["gains"] else None
        s.k_gain = _normal(g, (dim,), 600.0).add_(4096) if case["gains"] else None
        s.angles = _angles(case["positions"], case["rotated"] // 2)
        s.places = _integers(g, 0, case["positions"], (rows,))
        s.gain_shift, s.eps = 2, dim * dim
    elif kind == "choose":
        rows, vocab, history = case["rows"], case["vocab"], case["history"]
        # sums at 2^-23, and tokens of earlier steps: of the likely half, some of them often
        s.logits = torch.randn((rows, vocab), generator=g, device="cuda").mul_(2.5 * 2 ** 23).round_().long()
        r = random.Random(seed)
        s.counts = [history] + [r.randint(history // 2, history) for _ in range(rows - 1)]
        u = torch.rand((sum(s.counts),), generator=g, device="cuda")
        s.history = (u * u * vocab).int().clamp_(max=vocab - 1)
        s.bias_counts = [case["biases"]] + [r.randint(0, case["biases"]) for _ in range(rows - 1)]
        s.bias_tokens = _integers(g, 0, vocab, (sum(s.bias_counts),))
        s.bias_values = _integers(g, -(5 << 13), 5 << 13, (sum(s.bias_counts),))  # at 2^-13, in steps of 2^10
        s.bias_shift = 10
        # one bit a token; masks of the grammar's state, several sequences in the same
        s.masks = min(rows, 16) if case["masked"] else 0
        s.allowed = _integers(g, -(1 << 31), 1 << 31, (max(1, s.masks), (vocab + 31) // 32), torch.int64).int()
        s.mask_of = [r.randrange(s.masks) if s.masks else -1 for _ in range(rows)]
        s.repetition = [round(65536 * r.choice([1.0, 1.05, 1.1, 1.3])) for _ in range(rows)]
        s.frequency = [round(2 ** 23 * r.choice([0.0, 0.1, 0.5])) for _ in range(rows)]
        s.presence = [round(2 ** 23 * r.choice([0.0, 0.2, 0.6])) for _ in range(rows)]
    else:
        new, total = _lengths(case)
        rows, heads, kv_heads, dim, longest = sum(new), case["heads"], case["kv_heads"], case["dim"], max(total)
        s.new, s.total = new, total
        s.q = _normal(g, (rows, heads, dim), 1000.0)
        # the cache: tokens of earlier passes and of this one
        s.keys = _normal(g, (len(new), longest, kv_heads, dim), 1000.0)
        s.values = _normal(g, (len(new), longest, kv_heads, dim), 3000.0)
        if kind == "shared":
            s.prefix_k = _normal(g, (case["prefix"], kv_heads, dim), 1000.0)
            s.prefix_v = _normal(g, (case["prefix"], kv_heads, dim), 3000.0)
        s.table = _exponentials()
        s.shift = max(8, round(math.log2(math.sqrt(dim) * 1e6 / 1280.0)))
        first = np.concatenate([[0], np.cumsum(new)[:-1]])
        s.sequences = np.stack([np.arange(len(new)), first, np.array(new), np.array(total)], 1).astype(np.int64)
    return s


def prepare(case: dict, seed: int) -> _State:
    s = _inputs(case, seed)
    kind = case["kind"]
    if not own:
        if kind == "choose":
            # the plan: the row of each entry, and the rows' settings
            s.row = torch.repeat_interleave(torch.tensor(s.counts)).cuda()
            s.bias_row = torch.repeat_interleave(torch.tensor(s.bias_counts)).cuda()
            s.mask_of = torch.tensor(s.mask_of).cuda()
            s.settings = [torch.tensor(v).cuda()[:, None] for v in (s.repetition, s.frequency, s.presence)]
        elif kind != "rotate":
            # the plan: the place of each packed row
            s.seq = torch.cat([torch.full((m,), i) for i, m in enumerate(s.new)]).cuda()
            s.at = torch.cat([torch.arange(m) for m in s.new]).cuda()
            s.length = torch.tensor(s.total).cuda()
            s.before = torch.tensor([t - m for t, m in zip(s.total, s.new)]).cuda()
        return s
    r = s.r = _Resident()
    b = r.b
    if kind == "rotate":
        s.x, s.q_gain, s.k_gain = r.put(s.x), r.put(s.q_gain), r.put(s.k_gain)
        s.angles, s.places = (r.put(s.angles), r.put(s.places)) if case["rotated"] else (None, None)
        s.out, s.out_view = r.new((case["rows"], case["heads"] + case["kv_heads"], case["dim"]), np.int16)
    elif kind == "choose":
        from volta_mi355x import accel
        s.settings = np.zeros(case["rows"], accel.FIXED_CHOICE)
        s.settings["history_count"], s.settings["bias_count"] = s.counts, s.bias_counts
        for name, counts in (("history_first", s.counts), ("bias_first", s.bias_counts)):
            s.settings[name] = np.cumsum([0] + counts[:-1])
        s.settings["repetition"], s.settings["frequency"], s.settings["presence"] = s.repetition, s.frequency, s.presence
        s.settings["mask"] = s.mask_of
        s.logits, s.history, s.allowed = r.put(s.logits), r.put(s.history), r.put(s.allowed) if s.masks else None
        biased = sum(s.bias_counts) > 0
        s.bias_tokens, s.bias_values = (r.put(s.bias_tokens), r.put(s.bias_values)) if biased else (None, None)
        s.out, s.out_view = r.new((case["rows"],), np.int32)
        s.adjusted, s.adjusted_view = r.new((case["rows"], case["vocab"]), np.int64) if case["adjusted"] else (None, None)
    else:
        batch, longest = len(s.new), max(s.total)
        shared = kind == "shared"
        s.cache = b.fixed_kv_cache(batch + shared, case["kv_heads"], case["dim"],
                                   max(longest, case["prefix"] if shared else 0))
        r.kept.append((b.free_fixed_kv_cache, s.cache))
        fill = np.array([[i, i * longest, t, t] for i, t in enumerate(s.total)], np.int64)
        earlier = _Resident()
        b.fixed_kv_append_device(s.cache, earlier.put(s.keys), earlier.put(s.values), fill)
        if shared:  # in the slot behind the sequences'
            n = case["prefix"]
            b.fixed_kv_append_device(s.cache, earlier.put(s.prefix_k), earlier.put(s.prefix_v), [[batch, 0, n, n]])
            s.prefix_k = s.prefix_v = None
        b.synchronize()
        del earlier
        s.keys = s.values = None
        s.q, s.table = r.put(s.q), r.put(s.table)
        s.out, s.out_view = r.new((sum(s.new), case["heads"], case["dim"]), np.int16)
    b.synchronize()
    return s


# ---- one pass -------------------------------------------------------------------------------

def _rs(a: torch.Tensor, shift: int) -> torch.Tensor:
    return (a + (1 << (shift - 1))) >> shift if shift else a


def _sat(a: torch.Tensor) -> torch.Tensor:
    return a.clamp(-32768, 32767)


def _plain_rotate(s: _State):
    case = s.case
    heads, dim, pairs = case["heads"], case["dim"], case["rotated"] // 2
    h = s.x[:, :(heads + case["kv_heads"]) * dim].reshape(case["rows"], -1, dim).long()
    if case["gains"]:
        spread = dim * (h * h).sum(-1, keepdim=True) + s.eps
        root = spread.double().sqrt().long()
        root = torch.where(root * root > spread, root - 1, root)
        root = torch.where((root + 1) * (root + 1) <= spread, root + 1, root)
        below = root << s.gain_shift
        gain = torch.cat([s.q_gain.expand(heads, dim), s.k_gain.expand(case["kv_heads"], dim)]).long()
        h = _sat(torch.div(2 * dim * h * gain + below, 2 * below, rounding_mode="floor"))
    if pairs:
        turn = s.angles[s.places.long()].long()[:, None]
        c, d = turn[..., 0], turn[..., 1]
        if case["adjacent"]:
            a, b = h[..., 0:2 * pairs:2], h[..., 1:2 * pairs:2]
        else:
            a, b = h[..., :pairs], h[..., pairs:2 * pairs]
        a, b = _sat(_rs(a * c - b * d, 14)), _sat(_rs(a * d + b * c, 14))
        turned = torch.stack([a, b], -1).flatten(-2) if case["adjacent"] else torch.cat([a, b], -1)
        h = torch.cat([turned, h[..., 2 * pairs:]], -1)
    return h.to(torch.int16)


def _queries(s: _State, first: int, count: int):
    """Rows first .. first + count of each sequence: batch, key head, group x row, dim."""
    case = s.case
    q = torch.zeros(len(s.new), max(s.new), case["heads"], case["dim"], dtype=torch.int16, device="cuda")
    q[s.seq, s.at] = s.q
    q = q[:, first:first + count].double().view(len(s.new), count, case["kv_heads"], -1, case["dim"])
    return q.permute(0, 2, 3, 1, 4).reshape(len(s.new), case["kv_heads"], -1, case["dim"])


def _quotient(sums, total):
    return torch.div(2 * sums + total, (2 * total).clamp(min=1), rounding_mode="floor") * (total > 0)


def _plain_window(s: _State):
    case, batch = s.case, len(s.new)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    most, sinks = max(s.new), case["sinks"]
    window = min(case["window"], max(s.total))
    out = torch.zeros(batch, most, heads, dim, dtype=torch.int16, device="cuda")
    each = torch.arange(batch, device="cuda")[:, None]
    for first in range(0, most, QUERIES):
        count = min(QUERIES, most - first)
        p = s.before[:, None] + first + torch.arange(count, device="cuda")
        # keys that some of these rows may see: the sinks, then the rows' windows
        near = p[:, :1] - window + 1 + torch.arange(window + count - 1, device="cuda")
        j = torch.cat([torch.arange(sinks, device="cuda").expand(batch, sinks), near], 1)
        behind = torch.arange(j.shape[1], device="cuda") >= sinks
        there = (j >= 0) & (j < s.length[:, None]) & ~(behind & (j < sinks))
        seen = there[:, None] & (j[:, None] <= p[:, :, None]) & (~behind | (j[:, None] > p[:, :, None] - window))
        seen = seen[:, None, None]
        at = j.clamp(0, s.keys.shape[1] - 1)
        k = s.keys[each, at].double().permute(0, 2, 3, 1).contiguous()
        v = s.values[each, at].double().permute(0, 2, 1, 3).contiguous()
        z = (_queries(s, first, count) @ k).long().view(batch, kv_heads, -1, count, j.shape[1]) >> s.shift
        z = z.masked_fill_(~seen, -(1 << 60))
        z = (z.amax(-1, keepdim=True) - z).clamp_(max=ENTRIES - 1)
        e = s.table[z].long().masked_fill_(~seen, 0)
        sums = (e.double().view(batch, kv_heads, -1, j.shape[1]) @ v).long().view(batch, kv_heads, -1, count, dim)
        part = _quotient(sums, e.sum(-1, keepdim=True))
        out[:, first:first + count] = part.permute(0, 3, 1, 2, 4).reshape(batch, count, heads, dim)
    return out[s.seq, s.at]


def _plain_shared(s: _State):
    case, batch, most = s.case, len(s.new), max(s.new)
    heads, kv_heads, dim, longest = case["heads"], case["kv_heads"], case["dim"], s.keys.shape[1]
    group, prefix = heads // kv_heads, case["prefix"]
    q = _queries(s, 0, most)
    # the prefix: the rows of all sequences at once
    rows = q.transpose(0, 1).reshape(kv_heads, -1, dim)
    z0 = (rows @ s.prefix_k.double().permute(1, 2, 0).contiguous()).long()
    z0 = z0.view(kv_heads, batch, group, most, prefix).transpose(0, 1) >> s.shift
    k = s.keys.double().permute(0, 2, 3, 1).contiguous()
    z1 = (q @ k).long().view(batch, kv_heads, group, most, longest) >> s.shift
    place = torch.arange(longest, device="cuda")
    reach = s.before[:, None] + torch.arange(most, device="cuda")
    seen = ((place < s.length[:, None])[:, None] & (place <= reach[:, :, None]))[:, None, None]
    z1 = z1.masked_fill_(~seen, -(1 << 60))
    top = torch.maximum(z0.amax(-1, keepdim=True), z1.amax(-1, keepdim=True))
    e0 = s.table[(top - z0).clamp_(max=ENTRIES - 1)].long()
    e1 = s.table[(top - z1).clamp_(max=ENTRIES - 1)].long().masked_fill_(~seen, 0)
    total = e0.sum(-1, keepdim=True) + e1.sum(-1, keepdim=True)
    rows = e0.double().transpose(0, 1).reshape(kv_heads, -1, prefix)
    sums = (rows @ s.prefix_v.double().transpose(0, 1).contiguous()).view(kv_heads, batch, -1, dim).transpose(0, 1)
    v = s.values.double().permute(0, 2, 1, 3).contiguous()
    sums = sums + e1.double().view(batch, kv_heads, -1, longest) @ v
    out = _quotient(sums.long().view(batch, kv_heads, group, most, dim), total)
    return out.permute(0, 3, 1, 2, 4).reshape(batch, most, heads, dim)[s.seq, s.at].to(torch.int16)


def _plain_choose(s: _State):
    case = s.case
    rows, vocab = case["rows"], case["vocab"]
    repetition, frequency, presence = s.settings
    n = torch.zeros(rows * vocab, dtype=torch.int64, device="cuda")
    n = n.scatter_add_(0, s.row * vocab + s.history.long(), torch.ones_like(s.row)).view(rows, vocab)
    l = s.logits
    turned = torch.where(l < 0, _rs(l * repetition, 16),
                         torch.div((l << 17) + repetition, 2 * repetition, rounding_mode="floor"))
    l = torch.where(n > 0, turned - frequency * n - presence, l)
    if case["biases"]:
        added = torch.zeros(rows * vocab, dtype=torch.int64, device="cuda")
        added.scatter_add_(0, s.bias_row * vocab + s.bias_tokens.long(), s.bias_values.long() << s.bias_shift)
        l = l + added.view(rows, vocab)
    if s.masks:
        t = torch.arange(vocab, device="cuda")
        allowed = ((s.allowed[:, t // 32] >> (t % 32)) & 1).bool()[s.mask_of]
        l = l.masked_fill(~allowed, -(1 << 63))
    top = l.amax(1, keepdim=True)
    token = torch.where(l == top, torch.arange(vocab, device="cuda"), vocab).amin(1)
    token = torch.where(top[:, 0] == -(1 << 63), -1, token).to(torch.int32)
    return {"token": token, "logits": l} if case["adjusted"] else token


def run(s: _State):
    case, kind = s.case, s.case["kind"]
    if not own:
        return {"rotate": _plain_rotate, "window": _plain_window, "shared": _plain_shared,
                "choose": _plain_choose}[kind](s)
    b = s.r.b
    if kind == "rotate":
        b.fixed_rotate_device(s.x, case["rows"], case["heads"], case["dim"], kv_heads=case["kv_heads"],
                              x_stride=(case["heads"] + case["kv_heads"]) * case["dim"] + case["gap"], q_gain=s.q_gain,
                              k_gain=s.k_gain, gain_shift=s.gain_shift, eps=s.eps, angles=s.angles,
                              angle_rows=case["positions"], positions=s.places, rotated=case["rotated"],
                              adjacent=case["adjacent"], out=s.out)
        return s.out_view
    if kind == "choose":
        b.fixed_choose_device(s.logits, case["rows"], case["vocab"], s.settings, history=s.history,
                              bias_tokens=s.bias_tokens, bias_values=s.bias_values, bias_shift=s.bias_shift,
                              allowed=s.allowed, adjusted=s.adjusted, out=s.out)
        return {"token": s.out_view, "logits": s.adjusted_view} if case["adjusted"] else s.out_view
    if kind == "window":
        b.fixed_attention_device(s.q, s.cache, s.sequences, case["heads"], s.table, s.shift, window=case["window"],
                                 sinks=case["sinks"], out=s.out)
    else:
        b.fixed_attention_device(s.q, s.cache, s.sequences, case["heads"], s.table, s.shift,
                                 prefix=(len(s.new), case["prefix"]), out=s.out)
    return s.out_view


# ---- what a pass cannot do without ------------------------------------------------------------

def _seen(first: int, count: int, window: int, sinks: int) -> tuple[int, int]:
    """(pairs, keys read) of the rows at places first .. first + count of one sequence."""
    pairs = sum(min(p + 1, window) + max(0, min(sinks, p + 1 - window)) for p in range(first, first + count))
    near = max(0, first - window + 1)
    return pairs, first + count - near + min(sinks, near)


def work(case: dict) -> dict:
    """Each input read once and each output written once; multiply-adds of 16-bit integers as two operations."""
    kind = case["kind"]
    if kind == "rotate":
        n = case["rows"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        turns = 2 * min(case["rows"], case["positions"]) * case["rotated"] + 4 * case["rows"] * (case["rotated"] > 0)
        return {"bytes": 4 * n + turns + 4 * case["dim"] * case["gains"], "flops": (10 if case["gains"] else 6) * n}
    if kind == "choose":
        n = case["rows"] * case["vocab"]
        lists = case["rows"] * (3 * case["history"] + 4 * case["biases"])  # of 4 and 8 bytes, 0.75 and 0.5 full
        masks = min(case["rows"], 16) * ((case["vocab"] + 31) // 32) * 4 if case["masked"] else 0
        return {"bytes": (16 if case["adjusted"] else 8) * n + lists + masks + 4 * case["rows"], "flops": 2 * n}
    new, total = _lengths(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if kind == "window":
        seen = [_seen(t - m, m, case["window"], case["sinks"]) for m, t in zip(new, total)]
        pairs, keys = sum(a for a, _ in seen), sum(b for _, b in seen)
    else:
        pairs = sum(m * (case["prefix"] + t) - m * (m - 1) // 2 for m, t in zip(new, total))
        keys = case["prefix"] + sum(total)
    # queries and output, keys and values
    return {"bytes": 4 * sum(new) * heads * dim + 4 * kv_heads * dim * keys, "flops": 4 * dim * heads * pairs}


# ---- the definition, on the host ----------------------------------------------------------------

def _host(t):
    return None if t is None else t.cpu().numpy().astype(np.int64)


def _integer_product(a: np.ndarray, b: np.ndarray) -> np.ndarray:
    """a @ b of integers: the high and low halves of a apart, each product's sums under 2^53."""
    high, low = a >> 8, a & 255
    bf = b.astype(np.float64)
    return (np.rint(high.astype(np.float64) @ bf).astype(np.int64) << 8) + np.rint(low.astype(np.float64) @ bf).astype(
        np.int64)


def _rounded(a, shift: int):
    return np.floor_divide(a + ((1 << shift) >> 1), 1 << shift)


def _exact_rotate(case, s):
    heads, n, rotated = case["heads"], case["dim"], case["rotated"]
    y = _host(s.x)[:, :(heads + case["kv_heads"]) * n].reshape(case["rows"], -1, n)
    if case["gains"]:
        root = np.array([math.isqrt(int(v)) for v in (n * (y * y).sum(2) + s.eps).reshape(-1)], np.int64)
        root = root.reshape(y.shape[:2] + (1,)) << s.gain_shift
        gain = np.stack([_host(s.q_gain if h < heads else s.k_gain) for h in range(y.shape[1])])
        y = np.clip(np.floor_divide(2 * n * y * gain + root, 2 * root), -32768, 32767)
    out, angles, places = y.copy(), _host(s.angles), _host(s.places)
    for i in range(rotated // 2):
        first, second = (2 * i, 2 * i + 1) if case["adjacent"] else (i, i + rotated // 2)
        c, d = (angles[places, i, part][:, None] for part in (0, 1))
        out[..., first] = np.clip(_rounded(y[..., first] * c - y[..., second] * d, 14), -32768, 32767)
        out[..., second] = np.clip(_rounded(y[..., first] * d + y[..., second] * c, 14), -32768, 32767)
    return out.astype(np.int16)


def _exact_attention(q, k, v, seen, table, shift):
    """Rows of one head over the keys that ``seen`` marks."""
    z = np.floor_divide(_integer_product(q, k.T), 1 << shift)
    z[~seen] = -(1 << 60)
    e = table[np.minimum(z.max(1, keepdims=True) - z, len(table) - 1)]
    e[~seen] = 0
    den = e.sum(1, keepdims=True)
    return np.floor_divide(2 * _integer_product(e, v) + den, 2 * den)


def _exact_sequences(case, s):
    kind, heads, group = case["kind"], case["heads"], case["heads"] // case["kv_heads"]
    prefix = case["prefix"] if kind == "shared" else 0
    if heads * sum(m * (prefix + t) for m, t in zip(s.new, s.total)) > 4e8:
        return None  # minutes on the host
    q, table = _host(s.q), _host(s.table)
    out, row = np.zeros(q.shape, np.int16), 0
    for i, (m, t) in enumerate(zip(s.new, s.total)):
        k, v = _host(s.keys[i, :t]), _host(s.values[i, :t])
        if prefix:
            k, v = np.concatenate([_host(s.prefix_k), k]), np.concatenate([_host(s.prefix_v), v])
        j, p = np.arange(prefix + t)[None, :], (prefix + t - m + np.arange(m))[:, None]
        seen = j <= p
        if kind == "window":
            seen &= (j > p - case["window"]) | (j < case["sinks"])
        for h in range(heads):
            out[row:row + m, h] = _exact_attention(q[row:row + m, h], k[:, h // group], v[:, h // group], seen, table,
                                                   s.shift)
        row += m
    return out


def _exact_choose(case, s):
    logits, rows, vocab = _host(s.logits), case["rows"], case["vocab"]
    history, words = _host(s.history), _host(s.allowed) & 0xFFFFFFFF
    tokens, values = _host(s.bias_tokens), _host(s.bias_values)
    token, at, bias_at = np.zeros(rows, np.int32), 0, 0
    for i in range(rows):
        seen, counts = np.unique(history[at:at + s.counts[i]], return_counts=True)
        r = s.repetition[i]
        for t, n in zip(seen.tolist(), counts.tolist()):
            l = int(logits[i, t])
            l = (2 * l * r + 65536) // 131072 if l < 0 else (2 * l * 65536 + r) // (2 * r)
            logits[i, t] = l - s.frequency[i] * n - s.presence[i]
        for t, x in zip(tokens[bias_at:bias_at + s.bias_counts[i]].tolist(), values[bias_at:].tolist()):
            logits[i, t] += x * 2 ** s.bias_shift
        at, bias_at = at + s.counts[i], bias_at + s.bias_counts[i]
        if s.masks:
            bits = np.unpackbits(words[s.mask_of[i]].astype("<u4").view(np.uint8), bitorder="little")[:vocab]
            logits[i, bits == 0] = -(1 << 63)
        best = int(np.argmax(logits[i]))
        token[i] = -1 if logits[i, best] == -(1 << 63) else best
    return {"token": token, "logits": logits} if case["adjusted"] else token


def exact(case: dict, seed: int):
    s = _inputs(case, seed)
    return {"rotate": _exact_rotate, "choose": _exact_choose}.get(case["kind"], _exact_sequences)(case, s)
