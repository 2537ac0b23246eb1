"""Timed cases of the fixed-point model operators: the forward pass of the committed i16 weights.

A prover commits a model's quantised weights and then needs the trace of the
model's inference over them: embedding, norms, matrix products with their
epilogue, and attention over a cache of keys and values.  Everything is an
integer with an exact definition, so every correct implementation gives the
same values.

rs(a, s) is a / 2^s rounded to the nearest integer, halves up (a for s = 0);
sat clamps to 16 bits.

linear     acc = sum_k x[m, k] w[k, n] + (bias[n] << bias_shift); the sums
           themselves (``raw``), or h = sat(rs(acc, shift)), then table[h + 2^15],
           then sat(h + residual).
attention  keys and values of new tokens go to the cache; z = (q . k) >> shift,
           e = table[min(max z - z, len - 1)], out = sum e v / sum e rounded to
           the nearest integer, halves up.
norm       h = sat(x + residual); S = sum h, V = n sum h^2 - S^2 (rms: S = 0),
           R = floor(sqrt(V + eps)); y = sat((n h - S) gain / (R 2^shift), rounded
           to nearest, halves up, + bias).
embed      sat(rs(table[token] scale, shift) + positions[position]).

The plain forms work in 64 bits: products of 16-bit values summed over a row
pass 2^24, so 32-bit floating point cannot hold them, and 64-bit floating
point holds every sum here (under 2^53) exactly.
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
MOST_PRODUCTS = 16384 * 768 * 4096  # multiply-adds of the largest listed linear case
MOST_PAIRS = 16 * 8192 * 8192  # head x query x key places of the largest listed attention case


# ---- the cases ------------------------------------------------------------------------------

def listed() -> list[dict]:
    return [
        # One generated token through ffn_down (3072 x 768), with bias and the
        # residual stream: latency, and the reading of the weights.
        dict(name="linear_token", kind="linear", rows=1, k=3072, n=768, bias=True, table=False, residual=True,
             raw=False, gap=0),
        # An almost full context (1,023 of 1,024 positions) through ffn_up (768 x 3072) and the activation's table.
        dict(name="linear_prompt", kind="linear", rows=1023, k=768, n=3072, bias=True, table=True, residual=False,
             raw=False, gap=0),
        # Sums of the last position of seven sequences against the whole
        # vocabulary (50,257 tokens).
        dict(name="linear_logits", kind="linear", rows=7, k=768, n=50257, bias=False, table=False, residual=False,
             raw=True, gap=0),
        # Sixteen contexts through c_attn in its 768 x 4096 layout, rows read from a wider buffer.
        dict(name="linear_batch", kind="linear", rows=16384, k=768, n=4096, bias=True, table=False, residual=False,
             raw=False, gap=64),
        # One token of one sequence at the end of a full context, 12 heads of 64.
        dict(name="attention_token", kind="attention", batch=1, new=1, longest=1024, ragged=0, heads=12, kv_heads=12,
             dim=64, causal=True),
        # One token each of 64 sequences of different lengths, grouped heads.
        dict(name="attention_tokens", kind="attention", batch=64, new=1, longest=4095, ragged=5, heads=32, kv_heads=8,
             dim=128, causal=True),
        # Whole prompts of sixteen sequences of different lengths, packed, 12 heads of 64.
        dict(name="attention_prompts", kind="attention", batch=16, new=0, longest=1021, ragged=9, heads=12,
             kv_heads=12, dim=64, causal=True),
        # One long prompt, grouped heads of 128.
        dict(name="attention_long", kind="attention", batch=1, new=0, longest=8192, ragged=0, heads=16, kv_heads=4,
             dim=128, causal=True),
        # The norm before a generated token's block, without a residual.
        dict(name="norm_token", kind="norm", rows=1, cols=768, residual=False, rms=False),
        # The norm of sixteen contexts with the residual stream added and kept.
        dict(name="norm_batch", kind="norm", rows=16384, cols=768, residual=True, rms=False),
        # One generated token's embedding and position.
        dict(name="embed_token", kind="embed", rows=1, vocab=50257, cols=768, positions=1024, scaled=False),
        # Sixteen contexts of tokens, scaled.
        dict(name="embed_batch", kind="embed", rows=16384, vocab=50257, cols=768, positions=1024, scaled=True),
    ]


def _log(rng, lo: int, hi: int) -> int:
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(2.0 ** rng.uniform(math.log2(lo), math.log2(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["linear", "linear", "linear", "attention", "attention", "attention", "norm", "embed"])
    if kind == "linear":
        k, n = _log(rng, 16, 4096), _log(rng, 16, 50257)
        rows = _log(rng, 1, min(16384, MOST_PRODUCTS // (k * n)))
        raw = rng.random() < 0.2 and rows * n <= 1 << 26
        return dict(kind=kind, rows=rows, k=k, n=n, bias=rng.random() < 0.7, table=not raw and rng.random() < 0.4,
                    residual=not raw and rng.random() < 0.4, raw=raw, gap=rng.choice([0, 0, 8, 13]))
    if kind == "attention":
        kv_heads = rng.choice([1, 2, 4, 8, 12])
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
        dim = rng.choice([32, 40, 64, 64, 80, 96, 128, 128])
        batch = _log(rng, 1, 64)
        if rng.random() < 0.5:  # tokens over a cache
            new = _log(rng, 1, 8)
            most = min(8192, (1 << 28) // (batch * heads * dim * new), (1 << 29) // (batch * kv_heads * dim))
            longest = max(new, _log(rng, 1, most))
        else:  # whole prompts
            new, longest = 0, _log(rng, 1, max(1, min(8192, int(math.sqrt(MOST_PAIRS / (batch * heads))))))
        return dict(kind=kind, batch=batch, new=new, longest=longest, ragged=rng.randint(0, 1 << 20), heads=heads,
                    kv_heads=kv_heads, dim=dim, causal=rng.random() < 0.8)
    if kind == "norm":
        cols = _log(rng, 16, 8192)
        return dict(kind=kind, rows=_log(rng, 1, min(16384, (16384 * 768) // cols)), cols=cols,
                    residual=rng.random() < 0.6, rms=rng.random() < 0.4)
    cols = _log(rng, 16, 4096)
    return dict(kind=kind, rows=_log(rng, 1, min(16384, (16384 * 768) // cols)), vocab=_log(rng, 100, 50257), cols=cols,
                positions=_log(rng, 16, 1024), scaled=rng.random() < 0.5)


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
        if _backend is None:  # the one context that a prover process keeps, counting its calls without events
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
        buf, view = self.new(t.shape, {torch.int16: np.int16, torch.int32: np.int32}[t.dtype])
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


def _exponentials() -> torch.Tensor:
    """2^14 exp(-i / 640): 0 in the last entry."""
    i = np.arange(ENTRIES)
    return torch.from_numpy(np.rint(16384.0 * np.exp(-i / 640.0)).astype(np.int16)).cuda()


def _activation() -> torch.Tensor:
    """x Phi(x) over all 16-bit values at 2^-10."""
    x = np.arange(-32768, 32768) / 1024.0
    y = x * 0.5 * (1.0 + np.tanh(0.7978845608028654 * (x + 0.044715 * x ** 3)))
    return torch.from_numpy(np.rint(y * 1024.0).clip(-32768, 32767).astype(np.int16)).cuda()


def _inputs(case: dict, seed: int) -> _State:
    """What the case reads, as tensors: ``exact`` and both forms of ``run`` start from these."""
    s, kind = _State(), case["kind"]
    s.case = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if kind == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        s.x = _normal(g, (rows, k + case["gap"]), 1000.0)
        s.w = _normal(g, (k, n), 2000.0)
        s.bias = _normal(g, (n,), 2000.0) if case["bias"] else None
        s.bias_shift = 10
        s.residual = _normal(g, (rows, n), 3000.0) if case["residual"] else None
        s.table = _activation() if case["table"] else None
        s.shift = max(0, round(math.log2(math.sqrt(k) * 1000.0 * 2000.0 / 3000.0)))
    elif kind == "attention":
        new, total = _lengths(case)
        rows, heads, kv_heads, dim = sum(new), case["heads"], case["kv_heads"], case["dim"]
        s.new, s.total = new, total
        s.q = _normal(g, (rows, heads, dim), 1000.0)
        s.k = _normal(g, (rows, kv_heads, dim), 1000.0)
        s.v = _normal(g, (rows, kv_heads, dim), 3000.0)
        # the cache as it is before the pass: tokens of earlier passes
        past = max(t - m for t, m in zip(total, new))
        s.past_k = _normal(g, (len(new), past, kv_heads, dim), 1000.0)
        s.past_v = _normal(g, (len(new), past, kv_heads, dim), 3000.0)
        s.table = _exponentials()
        s.shift = max(8, round(math.log2(math.sqrt(dim) * 1e6 / 1280.0)))
        first = np.concatenate([[0], np.cumsum(new)[:-1]])
        s.sequences = np.stack([np.arange(len(new)), first, np.array(new), np.array(total)], 1).astype(np.int64)
    elif kind == "norm":
        rows, cols = case["rows"], case["cols"]
        s.x = _normal(g, (rows, cols), 2500.0)
        s.residual = _normal(g, (rows, cols), 5000.0) if case["residual"] else None
        s.gain = _normal(g, (cols,), 600.0).add_(4096)
        s.bias = None if case["rms"] else _normal(g, (cols,), 300.0)
        s.shift, s.eps = 2, cols * cols
    else:
        rows, vocab, cols = case["rows"], case["vocab"], case["cols"]
        s.tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
        s.places = torch.randint(0, case["positions"], (rows,), generator=g, device="cuda", dtype=torch.int32)
        s.words = _normal(g, (vocab, cols), 2000.0)
        s.where = _normal(g, (case["positions"], cols), 1000.0)
        s.scale, s.shift = (23170, 14) if case["scaled"] else (1, 0)
    return s


def prepare(case: dict, seed: int) -> _State:
    s = _inputs(case, seed)
    kind = case["kind"]
    if not own:
        if kind == "attention":
            # row-major caches with room for the pass's tokens, and the plan: the place of each packed row
            longest = max(s.total)
            room = longest - s.past_k.shape[1]
            pad = (0, 0, 0, 0, 0, room)
            s.past_k = torch.nn.functional.pad(s.past_k, pad)
            s.past_v = torch.nn.functional.pad(s.past_v, pad)
            s.seq = torch.cat([torch.full((m,), i) for i, m in enumerate(s.new)]).cuda()
            s.at = torch.cat([torch.arange(m) for m in s.new]).cuda()
            s.length = torch.tensor(s.total).cuda()
            s.before = torch.tensor([t - m for t, m in zip(s.total, s.new)]).cuda()
        return s
    r = s.r = _Resident()
    b = r.b
    if kind == "linear":
        w = r.put(s.w)
        s.weights = b.fixed_weights_device(w, case["k"], case["n"])
        r.kept.append((b.free_fixed_weights, s.weights))
        s.x, s.bias, s.residual, s.table = r.put(s.x), r.put(s.bias), r.put(s.residual), r.put(s.table)
        s.out, s.out_view = r.new((case["rows"], case["n"]), np.int64 if case["raw"] else np.int16)
    elif kind == "attention":
        capacity = max(s.total)
        s.cache = b.fixed_kv_cache(len(s.new), case["kv_heads"], case["dim"], capacity)
        r.kept.append((b.free_fixed_kv_cache, s.cache))
        past = s.past_k.shape[1]
        if past:
            fill = np.array([[i, i * past, past, past] for i in range(len(s.new))], np.int64)
            earlier = _Resident()
            b.fixed_kv_append_device(s.cache, earlier.put(s.past_k), earlier.put(s.past_v), fill)
            b.synchronize()
            del earlier
        s.past_k = s.past_v = None
        s.q, s.k, s.v, s.table = r.put(s.q), r.put(s.k), r.put(s.v), r.put(s.table)
        s.out, s.out_view = r.new((sum(s.new), case["heads"], case["dim"]), np.int16)
    elif kind == "norm":
        s.x, s.residual, s.gain, s.bias = r.put(s.x), r.put(s.residual), r.put(s.gain), r.put(s.bias)
        s.out, s.out_view = r.new((case["rows"], case["cols"]), np.int16)
        if s.residual is not None:
            s.total, s.total_view = r.new((case["rows"], case["cols"]), np.int16)
    else:
        s.tokens, s.places, s.words, s.where = r.put(s.tokens), r.put(s.places), r.put(s.words), r.put(s.where)
        s.out, s.out_view = r.new((case["rows"], case["cols"]), np.int16)
    b.synchronize()
    return s


# ---- one pass -------------------------------------------------------------------------------

def _rs(a: torch.Tensor, shift: int) -> torch.Tensor:
    return (a + (1 << (shift - 1))) >> shift if shift else a


def _sat(a: torch.Tensor) -> torch.Tensor:
    return a.clamp(-32768, 32767)


def _plain(s: _State):
    case, kind = s.case, s.case["kind"]
    if kind == "linear":
        acc = (s.x[:, :case["k"]].double() @ s.w.double()).long()
        if s.bias is not None:
            acc = acc + (s.bias.long() << s.bias_shift)
        if case["raw"]:
            return acc
        h = _sat(_rs(acc, s.shift))
        if s.table is not None:
            h = s.table[h + 32768].long()
        if s.residual is not None:
            h = _sat(h + s.residual.long())
        return h.to(torch.int16)
    if kind == "attention":
        heads, kv_heads, dim, batch = case["heads"], case["kv_heads"], case["dim"], len(s.new)
        group, longest, most = heads // kv_heads, s.past_k.shape[1], max(s.new)
        s.past_k[s.seq, s.at + s.before[s.seq]] = s.k
        s.past_v[s.seq, s.at + s.before[s.seq]] = s.v
        q = torch.zeros(batch, most, heads, dim, dtype=torch.float64, device="cuda")
        q[s.seq, s.at] = s.q.double()
        # rows of a key head's group together: batch, kv head, group x query
        q = q.view(batch, most, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, -1, dim)
        k = s.past_k.double().permute(0, 2, 3, 1).contiguous()
        v = s.past_v.double().permute(0, 2, 1, 3).contiguous()
        z = (q @ k).long().view(batch, kv_heads, group, most, longest) >> s.shift
        place = torch.arange(longest, device="cuda")
        allowed = (place < s.length[:, None])[:, None, None, None, :]
        if case["causal"]:
            reach = s.before[:, None] + torch.arange(most, device="cuda")
            allowed = allowed & (place <= reach[:, :, None])[:, None, None]
        z = z.masked_fill_(~allowed, -(1 << 60))
        z = (z.amax(-1, keepdim=True) - z).clamp_(max=ENTRIES - 1)
        e = s.table[z].long().masked_fill_(~allowed, 0)
        total = e.sum(-1, keepdim=True)
        sums = (e.double().view(batch, kv_heads, group * most, longest) @ v).long()
        sums = sums.view(batch, kv_heads, group, most, dim)
        out = torch.div(2 * sums + total, (2 * total).clamp(min=1), rounding_mode="floor") * (total > 0)
        out = out.permute(0, 3, 1, 2, 4).reshape(batch, most, heads, dim)
        return out[s.seq, s.at].to(torch.int16)
    if kind == "norm":
        h = s.x.long()
        if s.residual is not None:
            h = _sat(h + s.residual.long())
        n = case["cols"]
        first = 0 if case["rms"] else h.sum(1, keepdim=True)
        spread = n * (h * h).sum(1, keepdim=True) - first * first + s.eps
        root = spread.double().sqrt().long()
        root = torch.where(root * root > spread, root - 1, root)
        root = torch.where((root + 1) * (root + 1) <= spread, root + 1, root)
        below = root << s.shift
        y = torch.div(2 * (n * h - first) * s.gain.long() + below, 2 * below, rounding_mode="floor")
        if s.bias is not None:
            y = y + s.bias.long()
        y = _sat(y).to(torch.int16)
        return y if s.residual is None else {"y": y, "sum": h.to(torch.int16)}
    words = _rs(s.words[s.tokens.long()].long() * s.scale, s.shift)
    return _sat(words + s.where[s.places.long()].long()).to(torch.int16)


def run(s: _State):
    if not own:
        return _plain(s)
    case, kind, b = s.case, s.case["kind"], s.r.b
    if kind == "linear":
        b.fixed_linear_device(s.x, case["rows"], s.weights, s.shift, x_stride=case["k"] + case["gap"], bias=s.bias,
                              bias_shift=s.bias_shift, table=s.table, residual=s.residual, raw=case["raw"], out=s.out)
        return s.out_view
    if kind == "attention":
        # the cache then holds the pass's keys and values as given; what is computed from it is returned
        b.fixed_kv_append_device(s.cache, s.k, s.v, s.sequences)
        b.fixed_attention_device(s.q, s.cache, s.sequences, case["heads"], s.table, s.shift, causal=case["causal"],
                                 out=s.out)
        return s.out_view
    if kind == "norm":
        if s.residual is None:
            b.fixed_norm_device(s.x, case["rows"], case["cols"], s.gain, s.shift, s.eps, bias=s.bias, rms=case["rms"],
                                out=s.out)
            return s.out_view
        b.fixed_norm_device(s.x, case["rows"], case["cols"], s.gain, s.shift, s.eps, bias=s.bias, rms=case["rms"],
                            residual=s.residual, sum_out=s.total, out=s.out)
        return {"y": s.out_view, "sum": s.total_view}
    b.fixed_embed_device(s.tokens, case["rows"], s.words, case["vocab"], case["cols"], scale=s.scale, shift=s.shift,
                         positions=s.places, position_table=s.where, position_rows=case["positions"], out=s.out)
    return s.out_view


# ---- what a pass cannot do without ------------------------------------------------------------

def work(case: dict) -> dict:
    """Each input read once and each output written once; multiply-adds of 16-bit integers as two operations."""
    kind = case["kind"]
    if kind == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        size = 2 * m * k + 2 * k * n + (8 if case["raw"] else 2) * m * n
        size += 2 * n * case["bias"] + 2 * m * n * case["residual"] + (1 << 17) * case["table"]
        return {"bytes": size, "flops": 2 * m * k * n}
    if kind == "attention":
        new, total = _lengths(case)
        heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
        pairs = sum(m * t - (m * (m - 1) // 2 if case["causal"] else 0) for m, t in zip(new, total))
        # queries and output; keys and values of all tokens read, those of the new ones also written
        size = 4 * sum(new) * heads * dim + 4 * kv_heads * dim * (sum(total) + sum(new))
        return {"bytes": size, "flops": 4 * dim * heads * pairs}
    if kind == "norm":
        size = 2 * case["rows"] * case["cols"]
        return {"bytes": size * (4 if case["residual"] else 2) + 4 * case["cols"],
                "flops": 10 * case["rows"] * case["cols"]}
    return {"bytes": 6 * case["rows"] * case["cols"] + 8 * case["rows"], "flops": 2 * case["rows"] * case["cols"]}


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


def exact(case: dict, seed: int):
    kind = case["kind"]
    s = _inputs(case, seed)
    if kind == "linear":
        acc = _integer_product(_host(s.x)[:, :case["k"]], _host(s.w))
        if s.bias is not None:
            acc += _host(s.bias) * (1 << s.bias_shift)
        if case["raw"]:
            return acc
        h = np.clip(_rounded(acc, s.shift), -32768, 32767)
        if s.table is not None:
            h = _host(s.table)[h + 32768]
        if s.residual is not None:
            h = np.clip(h + _host(s.residual), -32768, 32767)
        return h.astype(np.int16)
    if kind == "attention":
        heads, group, dim = case["heads"], case["heads"] // case["kv_heads"], case["dim"]
        new, total = s.new, s.total
        if heads * sum(m * t for m, t in zip(new, total)) > 4e8:
            return None  # minutes on the host
        q, k, v = _host(s.q), _host(s.k), _host(s.v)
        past_k, past_v, table = _host(s.past_k), _host(s.past_v), _host(s.table)
        out, row = np.zeros(q.shape, np.int16), 0
        for i, (m, t) in enumerate(zip(new, total)):
            keys = np.concatenate([past_k[i, :t - m], k[row:row + m]])
            values = np.concatenate([past_v[i, :t - m], v[row:row + m]])
            hidden = np.arange(t)[None, :] > (t - m + np.arange(m))[:, None] if case["causal"] else np.zeros((m, t), bool)
            for h in range(heads):
                z = np.floor_divide(_integer_product(q[row:row + m, h], keys[:, h // group].T), 1 << s.shift)
                z[hidden] = -(1 << 60)
                e = table[np.minimum(z.max(1, keepdims=True) - z, len(table) - 1)]
                e[hidden] = 0
                den = e.sum(1, keepdims=True)
                num = _integer_product(e, values[:, h // group])
                out[row:row + m, h] = np.floor_divide(2 * num + den, 2 * den)
            row += m
        return out
    if kind == "norm":
        h = _host(s.x)
        if s.residual is not None:
            h = np.clip(h + _host(s.residual), -32768, 32767)
        n = case["cols"]
        centre = n * h if case["rms"] else n * h - h.sum(1, keepdims=True)
        spread = n * (h * h).sum(1) - (0 if case["rms"] else h.sum(1) ** 2) + s.eps
        root = np.array([math.isqrt(int(x)) for x in spread], np.int64)[:, None] << s.shift
        y = np.floor_divide(2 * centre * _host(s.gain) + root, 2 * root)
        if s.bias is not None:
            y = y + _host(s.bias)
        y = np.clip(y, -32768, 32767).astype(np.int16)
        return y if s.residual is None else {"y": y, "sum": h.astype(np.int16)}
    words = _rounded(_host(s.words)[_host(s.tokens)] * s.scale, s.shift)
    return np.clip(words + _host(s.where)[_host(s.places)], -32768, 32767).astype(np.int16)
