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
the residual added in its epilogue.
"""
from __future__ import annotations

from dataclasses import dataclass

import numpy as np

from .accel import Backend, DeviceBuffer, InvalidInput


@dataclass(frozen=True)
class FixedConfig:
    """Sizes, and the binary points that the shifts keep.  Activations are at 2^-act_bits, and so is what is added to
    them: norm biases and wpe.  Weights, wte among them, and the biases of products are at 2^-weight_bits, norm gains at
    2^-gain_bits; `bits` gives each tensor's."""
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

    def __post_init__(self):
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
        out = {"wte": (self.vocab, self.width), "wpe": (self.positions, self.width), "norm.gain": (self.width,),
               "norm.bias": (self.width,)}
        for i in range(self.layers):
            for name, k, n in (("qkv", self.width, self.qkv_width), ("proj", self.width, self.width),
                               ("up", self.width, self.hidden), ("down", self.hidden, self.width)):
                out[f"h{i}.{name}"], out[f"h{i}.{name}.bias"] = (k, n), (n,)
            for name in ("norm1", "norm2"):
                out[f"h{i}.{name}.gain"] = out[f"h{i}.{name}.bias"] = (self.width,)
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
        self.lengths = [0] * slots
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
        """Forgets a slot's sequence."""
        self.lengths[slot] = 0

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
        after = [self.lengths[s] + n for s, n in zip(slots, counts)]
        if max(after) > c.positions:
            raise InvalidInput("a sequence is longer than the model's positions")
        first = np.concatenate([[0], np.cumsum(counts)[:-1]])
        seqs = np.stack([slots, first, counts, after], 1).astype(np.int64)
        b.upload_into(self._tokens, 0, np.concatenate(prompts))
        b.upload_into(self._places, 0, np.concatenate([np.arange(a - n, a, dtype=np.int32)
                                                       for a, n in zip(after, counts)]))
        h, n, part = self._h, self._n, self._part
        b.fixed_embed_device(self._tokens, rows, self.tensors["wte"], c.vocab, c.width,
                             scale=c.embed_scale, shift=c.embed_shift, positions=self._places,
                             position_table=self.tensors["wpe"], position_rows=c.positions, out=h)
        for i in range(c.layers):
            self._norm(f"h{i}.norm1", h, rows)
            self._linear(f"h{i}.qkv", n, rows, self._qkv)
            b.fixed_kv_append_device(self._caches[i], self._qkv, self._qkv, seqs, k_offset=c.width,
                                     k_stride=c.qkv_width, v_offset=c.width + c.kv_width, v_stride=c.qkv_width)
            b.fixed_attention_device(self._qkv, self._caches[i], seqs, c.heads, self._exp, c.score_shift,
                                     q_stride=c.qkv_width, out=n)
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

    def generate(self, prompt, count: int, slot: int = 0) -> list[int]:
        """The `count` tokens of the largest logits (the lowest index of equal ones) after the prompt."""
        out: list[int] = []
        tokens = list(prompt)
        for _ in range(count):
            out.append(int(np.argmax(self.step([tokens], [slot])[0])))
            tokens = out[-1:]
        return out
