"""The committed model's forward pass: a decoder over resident i16 tensors.

The tensors that `ligero.commit_resident_from_device` commits are the ones that
run here: the same resident buffers, in fixed point, with exact sums and defined
roundings, so an inference gives the same values however its tokens are batched
(a whole prompt at once or token by token) and on whatever GPU.  Logits are what
it returns; a layer's values are overwritten by the next.  The roundings and
tables are this library's own: no reference output fixes them (parity unpinned).

    model = FixedDecoder(backend, config, tensors, slots=4)
    logits = model.step([prompt_a, prompt_b], [0, 1])     # i64 sums, a row a sequence
    tokens = model.generate(prompt, 20)

A block is: norm, query-key-value product, attention over the slots' cache,
output product; its sum with the residual stream is taken in the second norm;
then the hidden product with the activation's table and the product back, with
the residual added in its epilogue.  With head norms or rotary positions the
queries and keys are normed and rotated in one pass before the keys are kept; with
a window a token sees the last of its keys and the sequence's first ones.

    model.share(instructions, slot=3)       # the other slots' sequences begin with it, held once
    model.generate(prompt, 20, repetition=1.1, bias={7: -2.0}, allowed=mask)
"""
from __future__ import annotations

from collections.abc import Iterable
from dataclasses import dataclass
from numbers import Real

import numpy as np

from .accel import FIXED_CHOICE, Backend, DeviceBuffer, InvalidInput


@dataclass(frozen=True)
class FixedConfig:
    """Sizes, and the binary points that the shifts keep.  Activations are at 2^-act_bits, and so is what is added to
    them: norm biases and wpe.  Weights, wte among them, and the biases of products are at 2^-weight_bits, norm gains at
    2^-gain_bits; `bits` gives each tensor's.

    Positions are learned (wpe) or, with `rotary`, turn the first `rotary` places of each query and key, in pairs of
    places half of them apart or adjacent.  `head_norm` gives queries and keys an RMS norm of each head before that.
    `window` (0: none) bounds what a token sees to the last keys, its own among them, and the sequence's first `sinks`;
    a slot keeps `positions` tokens all the same."""
    layers: int
    heads: int
    kv_heads: int
    dim: int          # of a head
    hidden: int
    vocab: int
    positions: int
    act_bits: int = 10
    weight_bits: int = 13
    gain_bits: int = 12
    eps: float = 1e-5
    rotary: int = 0
    rotary_base: float = 10000.0
    adjacent: bool = False
    head_norm: bool = False
    window: int = 0
    sinks: int = 0

    def __post_init__(self):
        if not 0 <= self.rotary <= self.dim or self.rotary % 2 or not self.rotary_base > 0:
            raise InvalidInput("rotary is an even number of a head's places")
        if self.window < 0 or self.sinks < 0 or (self.sinks and not self.window):
            raise InvalidInput("sinks come with a window")
        # 15: past it the exponential table no longer reaches down to 0; the others are the operators' shifts
        if not 0 <= self.act_bits <= 15 or not 0 <= self.weight_bits <= 46:
            raise InvalidInput("act_bits goes from 0 to 15, weight_bits from 0 to 46")
        if not 0 <= self.gain_bits - self.act_bits <= 15:
            raise InvalidInput("gain_bits is act_bits to act_bits + 15")

    @property
    def width(self) -> int:
        return self.heads * self.dim

    @property
    def kv_width(self) -> int:
        return self.kv_heads * self.dim

    @property
    def qkv_width(self) -> int:
        return self.width + 2 * self.kv_width

    @property
    def norm_eps(self) -> int:
        """eps in the norm's units: cols^2 times a variance at 2^-2 act_bits."""
        return max(1, round(self.eps * self.width ** 2 * 4 ** self.act_bits))

    @property
    def head_eps(self) -> int:
        """eps in the units of a head's norm."""
        return max(1, round(self.eps * self.dim ** 2 * 4 ** self.act_bits))

    @property
    def embed_scale(self) -> int:
        """With embed_shift, takes wte's rows from 2^-weight_bits to 2^-act_bits."""
        return 1 << max(0, self.act_bits - self.weight_bits)

    @property
    def embed_shift(self) -> int:
        return max(0, self.weight_bits - self.act_bits)

    @property
    def score_shift(self) -> int:
        """Leaves scores in steps of about 1/640 after the division by sqrt(dim)."""
        return min(24, max(8, round(2 * self.act_bits + np.log2(np.sqrt(self.dim) / 640))))

    def shapes(self) -> dict[str, tuple[int, ...]]:
        """Names and shapes of the tensors a model is made of (matrices k x n, as committed)."""
        out = {"wte": (self.vocab, self.width), "norm.gain": (self.width,), "norm.bias": (self.width,)}
        if not self.rotary:
            out["wpe"] = (self.positions, self.width)
        for i in range(self.layers):
            for name, k, n in (("qkv", self.width, self.qkv_width), ("proj", self.width, self.width),
                               ("up", self.width, self.hidden), ("down", self.hidden, self.width)):
                out[f"h{i}.{name}"], out[f"h{i}.{name}.bias"] = (k, n), (n,)
            for name in ("norm1", "norm2"):
                out[f"h{i}.{name}.gain"] = out[f"h{i}.{name}.bias"] = (self.width,)
            if self.head_norm:
                out[f"h{i}.q_norm.gain"] = out[f"h{i}.k_norm.gain"] = (self.dim,)
        return out

    def bits(self, name: str) -> int:
        """The binary point of tensor `name`: a value v is held as round(v 2^bits)."""
        if name not in self.shapes():
            raise InvalidInput(f"the model has no tensor {name}")
        if name.endswith(".gain"):
            return self.gain_bits
        norm_bias = name.endswith(".bias") and name.split(".")[-2].startswith("norm")
        return self.act_bits if norm_bias or name == "wpe" else self.weight_bits


def activation_table(act_bits: int) -> np.ndarray:
    """65,536 entries of x Phi(x), the tanh form, for 16-bit x at 2^-act_bits."""
    x = np.arange(-32768, 32768) / float(1 << act_bits)
    y = x * 0.5 * (1.0 + np.tanh(0.7978845608028654 * (x + 0.044715 * x ** 3)))
    return np.rint(y * (1 << act_bits)).clip(-32768, 32767).astype(np.int16)


def exponential_table(config: FixedConfig, entries: int = 8192) -> np.ndarray:
    """2^14 exp(-d step) for d below `entries`, with the step that score_shift leaves; 0 in the last."""
    step = 2.0 ** (config.score_shift - 2 * config.act_bits) / np.sqrt(config.dim)
    table = np.rint(16384.0 * np.exp(-np.arange(entries) * step)).astype(np.uint16)
    table[-1] = 0
    return table


def rotation_table(config: FixedConfig) -> np.ndarray:
    """positions x rotary / 2 pairs (cos, sin) at 2^-14 of position / rotary_base^(2 i / rotary)."""
    turns = config.rotary_base ** (-np.arange(config.rotary // 2) / max(1, config.rotary // 2))
    angles = np.arange(config.positions)[:, None] * turns
    return np.rint(16384.0 * np.stack([np.cos(angles), np.sin(angles)], -1)).astype(np.int16)


class FixedDecoder:
    """A decoder with `slots` sequences of up to config.positions tokens and `rows` tokens a step (default: all)."""

    def __init__(self, backend: Backend, config: FixedConfig, tensors: dict[str, DeviceBuffer], slots: int = 1,
                 rows: int | None = None):
        c = self.config = config
        self.backend, self.slots = backend, slots
        self.rows = rows or slots * c.positions
        for name, shape in c.shapes().items():
            if name not in tensors or tensors[name].len < int(np.prod(shape)) or tensors[name].dtype != np.int16:
                raise InvalidInput(f"tensor {name} must hold {shape} i16")
        self.tensors = tensors
        self.lengths = [0] * slots  # without the shared prefix
        self.prefix: tuple[int, int] | None = None  # its slot and tokens
        self._bufs: list[DeviceBuffer] = []
        self._packed, self._caches = {}, []
        try:
            for name, shape in c.shapes().items():
                if len(shape) == 2 and name != "wpe":
                    vocab = name == "wte"  # wte's rows are the logits' columns
                    k, n = (c.width, c.vocab) if vocab else shape
                    self._packed[name] = backend.fixed_weights_device(tensors[name], k, n, transposed=vocab)
            for _ in range(c.layers):
                self._caches.append(backend.fixed_kv_cache(slots, c.kv_heads, c.dim, c.positions))
            self._act = self._keep(backend.upload_device(activation_table(c.act_bits)))
            self._exp = self._keep(backend.upload_device(exponential_table(c)))
            self._tokens, self._places = (self._keep(backend.alloc_device(self.rows, np.int32)) for _ in range(2))
            self._h, self._n, self._part = (self._keep(backend.alloc_device(self.rows * c.width, np.int16))
                                            for _ in range(3))
            self._qkv = self._keep(backend.alloc_device(self.rows * c.qkv_width, np.int16))
            self._up = self._keep(backend.alloc_device(self.rows * c.hidden, np.int16))
            self._logits = self._keep(backend.alloc_device(slots * c.vocab, np.int64))
            self._angles = self._keep(backend.upload_device(rotation_table(c).reshape(-1))) if c.rotary else None
            self._history = self._keep(backend.alloc_device(c.positions + 1, np.int32))
            self._allowed = self._keep(backend.alloc_device((c.vocab + 31) // 32, np.uint32))
            self._next = self._keep(backend.alloc_device(1, np.int32))
        except Exception:
            self.close()
            raise

    def _keep(self, buf: DeviceBuffer) -> DeviceBuffer:
        self._bufs.append(buf)
        return buf

    def close(self) -> None:
        """Frees what the decoder allocated (not the tensors)."""
        for w in self._packed.values():
            self.backend.free_fixed_weights(w)
        for cache in self._caches:
            self.backend.free_fixed_kv_cache(cache)
        for buf in self._bufs:
            self.backend.free_device(buf)
        self._packed, self._caches, self._bufs = {}, [], []

    def reset(self, slot: int) -> None:
        """Forgets a slot's sequence (not the prefix that the slots share)."""
        if self.prefix is not None and slot == self.prefix[0]:
            raise InvalidInput("the slot holds the shared prefix")
        self.lengths[slot] = 0

    def share(self, prompt, slot: int) -> None:
        """Runs `prompt` in `slot`, in steps of the decoder's rows, and makes its tokens the beginning of the sequences of
        all other slots, which are empty.  They are kept once, and attention reads them once for all sequences of a step."""
        if self.config.window:
            raise InvalidInput("a window and a shared prefix do not go together")
        if self.prefix is not None or any(self.lengths):
            raise InvalidInput("a prefix is shared before any sequence begins")
        tokens = self._prompt(prompt)
        if not 0 <= slot < self.slots:
            raise InvalidInput("slot is outside the decoder's")
        if not 0 < len(tokens) <= self.config.positions:
            raise InvalidInput("a prefix holds one token to the model's positions")
        try:
            for at in range(0, len(tokens), self.rows):
                self.step_device([tokens[at:at + self.rows]], [slot])
        except Exception:
            self.lengths[slot] = 0
            raise
        self.prefix = (slot, len(tokens))

    def unshare(self) -> None:
        """Forgets the shared prefix and all sequences."""
        self.prefix = None
        self.lengths = [0] * self.slots

    def _linear(self, name: str, x: DeviceBuffer, rows: int, out: DeviceBuffer, **kw) -> None:
        c = self.config
        self.backend.fixed_linear_device(x, rows, self._packed[name], c.weight_bits, bias=self.tensors[name + ".bias"],
                                         bias_shift=c.act_bits, out=out, **kw)

    def _norm(self, name: str, x: DeviceBuffer, rows: int, **kw) -> None:
        c = self.config
        # n h - S over R is the normalised value; gain / 2^(gain_bits - act_bits) leaves it at 2^-act_bits
        self.backend.fixed_norm_device(x, rows, c.width, self.tensors[name + ".gain"], c.gain_bits - c.act_bits,
                                       c.norm_eps, bias=self.tensors[name + ".bias"], out=self._n, **kw)

    def _prompt(self, prompt) -> np.ndarray:
        """A prompt's tokens, checked before they become i32: a larger integer would turn into another token."""
        t = np.asarray(prompt)
        if t.ndim != 1 or t.size and t.dtype.kind not in "biu":
            raise InvalidInput("a prompt is one row of integer tokens")
        if t.size and (t.min() < 0 or t.max() >= self.config.vocab):
            raise InvalidInput("token is outside the vocabulary")
        return t.astype(np.int32)

    def step_device(self, prompts, slots) -> DeviceBuffer:
        """Appends each prompt's tokens to its slot; the logits' i64 sums after its last token, a row a prompt."""
        c, b = self.config, self.backend
        prompts = [self._prompt(p) for p in prompts]
        counts = [len(p) for p in prompts]
        rows = sum(counts)
        if len(slots) != len(counts) or not counts or min(counts) == 0 or rows > self.rows or len(set(slots)) != len(slots):
            raise InvalidInput("a step takes one non-empty prompt for each of its slots, within the decoder's rows")
        if min(slots) < 0 or max(slots) >= self.slots:
            raise InvalidInput("slot is outside the decoder's")
        if self.prefix is not None and self.prefix[0] in slots:
            raise InvalidInput("the slot holds the shared prefix")
        before = self.prefix[1] if self.prefix is not None else 0
        after = [self.lengths[s] + n for s, n in zip(slots, counts)]
        if before + max(after) > c.positions:
            raise InvalidInput("a sequence is longer than the model's positions")
        first = np.concatenate([[0], np.cumsum(counts)[:-1]])
        seqs = np.stack([slots, first, counts, after], 1).astype(np.int64)
        b.upload_into(self._tokens, 0, np.concatenate(prompts))
        b.upload_into(self._places, 0, np.concatenate([np.arange(before + a - n, before + a, dtype=np.int32)
                                                       for a, n in zip(after, counts)]))
        h, n, part = self._h, self._n, self._part
        learned = {} if c.rotary else dict(positions=self._places, position_table=self.tensors["wpe"],
                                           position_rows=c.positions)
        b.fixed_embed_device(self._tokens, rows, self.tensors["wte"], c.vocab, c.width, scale=c.embed_scale,
                             shift=c.embed_shift, out=h, **learned)
        heads = dict(kv_heads=c.kv_heads, x_stride=c.qkv_width, out=self._qkv, out_stride=c.qkv_width)
        if c.rotary:
            heads.update(angles=self._angles, angle_rows=c.positions, positions=self._places, rotated=c.rotary,
                         adjacent=c.adjacent)
        for i in range(c.layers):
            self._norm(f"h{i}.norm1", h, rows)
            self._linear(f"h{i}.qkv", n, rows, self._qkv)
            if c.head_norm:
                heads.update(q_gain=self.tensors[f"h{i}.q_norm.gain"], k_gain=self.tensors[f"h{i}.k_norm.gain"],
                             gain_shift=c.gain_bits - c.act_bits, eps=c.head_eps)
            if c.head_norm or c.rotary:
                b.fixed_rotate_device(self._qkv, rows, c.heads, c.dim, **heads)
            b.fixed_kv_append_device(self._caches[i], self._qkv, self._qkv, seqs, k_offset=c.width,
                                     k_stride=c.qkv_width, v_offset=c.width + c.kv_width, v_stride=c.qkv_width)
            b.fixed_attention_device(self._qkv, self._caches[i], seqs, c.heads, self._exp, c.score_shift,
                                     q_stride=c.qkv_width, window=c.window, sinks=c.sinks, prefix=self.prefix, out=n)
            self._linear(f"h{i}.proj", n, rows, part)
            self._norm(f"h{i}.norm2", part, rows, residual=h, sum_out=h)
            self._linear(f"h{i}.up", n, rows, self._up, table=self._act)
            self._linear(f"h{i}.down", self._up, rows, h, residual=h)
        self._norm("norm", h, rows)
        if rows == len(counts):
            b.fixed_linear_device(n, rows, self._packed["wte"], raw=True, out=self._logits)
        else:
            for i, (at, count) in enumerate(zip(first, counts)):
                b.fixed_linear_device(n, 1, self._packed["wte"], raw=True, x_offset=int(at + count - 1) * c.width,
                                      out=self._logits, out_offset=i * c.vocab)
        for s, length in zip(slots, after):
            self.lengths[s] = length
        return self._logits

    def step(self, prompts, slots) -> np.ndarray:
        """step_device's logits on the host: prompts x vocab i64."""
        out = self.step_device(prompts, slots)
        return self.backend.download_device(out, 0, len(slots) * self.config.vocab).reshape(len(slots), -1)

    def _fixed(self, value: float) -> int:
        """A number in the logits' units."""
        return round(value * 2.0 ** (self.config.act_bits + self.config.weight_bits))

    def _words(self, allowed) -> np.ndarray:
        """A mask of the vocabulary as words of 32 bits."""
        a = np.asarray(allowed)
        if a.dtype != np.bool_ or a.shape != (self.config.vocab,):
            raise InvalidInput("allowed is a truth value for each token")
        return np.packbits(np.pad(a, (0, -len(a) % 32)), bitorder="little").view("<u4")

    def generate(self, prompt, count: int, slot: int = 0, *, repetition: float = 1.0, frequency: float = 0.0,
                 presence: float = 0.0, bias: dict[int, float] | None = None, allowed=None) -> list[int]:
        """The `count` tokens of the largest logits (the lowest index of equal ones) after the prompt, any iterable of
        tokens.

        The logit of a token that the prompt and the answer hold n > 0 times is divided by `repetition` (multiplied, if
        negative) and lowered by frequency n + presence: all three count the prompt's tokens, and none counts those that
        the slot held before or a shared prefix.  `bias` is added to its tokens' logits, to the nearest 2^-13 (or step of
        the logits, if that is coarser).  `allowed`: a truth value for each token, or a function that gives them for the
        answer so far; where it allows nothing, the answer ends."""
        c, b = self.config, self.backend
        if count <= 0:
            return []
        if not 0 <= slot < self.slots:
            raise InvalidInput("slot is outside the decoder's")
        choice = np.zeros(1, FIXED_CHOICE)
        unit = c.act_bits + c.weight_bits
        scale = repetition * 65536.0
        limit = 2.0 ** (62 - unit)
        if not 1 <= scale <= 2 ** 32 - 1 or not abs(frequency) < limit or not abs(presence) < limit:
            raise InvalidInput("a penalty is out of range")
        choice["repetition"], choice["mask"] = round(scale), -1
        choice["frequency"], choice["presence"] = self._fixed(frequency), self._fixed(presence)
        # biases at 2^-13, or as finely as the logits are; the operator shifts them by 46 at most
        bits = max(min(13, unit), unit - 46)
        bias = bias or {}
        if any(not isinstance(t, Real) or not 0 <= t < c.vocab or t != int(t) for t in bias):
            raise InvalidInput("a bias is for a token of the vocabulary")
        if any(not abs(v) < 2.0 ** (31 - bits) - 1 for v in bias.values()):
            raise InvalidInput("a bias is out of range")
        penalized = repetition != 1.0 or frequency or presence
        if not isinstance(prompt, np.ndarray) and isinstance(prompt, Iterable):
            prompt = list(prompt)  # of an iterator or a set too
        tokens = self._prompt(prompt)
        before = self.lengths[slot] + (self.prefix[1] if self.prefix is not None else 0)
        if before + len(tokens) + count > c.positions + 1:
            raise InvalidInput("a sequence is longer than the model's positions")
        held: list[DeviceBuffer] = []
        out: list[int] = []
        try:
            lists = {}
            if bias:
                held += [b.upload_device(np.array(list(bias), np.int32)),
                         b.upload_device(np.rint(np.array(list(bias.values())) * 2.0 ** bits).astype(np.int32))]
                lists = dict(bias_tokens=held[0], bias_values=held[1], bias_shift=unit - bits)
                choice["bias_count"] = len(bias)
            if penalized:
                b.upload_into(self._history, 0, tokens)
                choice["history_count"] = len(tokens)
                lists["history"] = self._history
            if allowed is not None:
                lists["allowed"] = self._allowed
                choice["mask"] = 0
                if not callable(allowed):
                    b.upload_into(self._allowed, 0, self._words(allowed))
            for _ in range(count):
                if callable(allowed):
                    b.upload_into(self._allowed, 0, self._words(allowed(list(out))))
                logits = self.step_device([tokens], [slot])
                b.fixed_choose_device(logits, 1, c.vocab, choice, out=self._next, **lists)
                token = int(b.download_device(self._next)[0])
                if token < 0:
                    break
                out.append(token)
                tokens = out[-1:]
                if penalized:
                    b.upload_into(self._history, int(choice["history_count"][0]), np.array(tokens, np.int32))
                    choice["history_count"] += 1
        finally:
            for buf in held:
                b.free_device(buf)
        return out
