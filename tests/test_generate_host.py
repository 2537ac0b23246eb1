"""What FixedDecoder.generate and share do on the host: a decoder without a GPU, whose steps and choices are written down."""
import numpy as np
import pytest
from volta_mi355x import InvalidInput, forward

SIZES = dict(layers=1, heads=2, kv_heads=1, dim=8, hidden=16, vocab=50, positions=24)


class Buffer:
    def __init__(self, values):
        self.values = np.array(values)


class Library:
    """The calls of `generate` on a backend: the token chosen is one more than the last of the step."""

    def __init__(self):
        self.choices = []

    def upload_device(self, values):
        return Buffer(values)

    def upload_into(self, buf, offset, values):
        buf.values[offset:offset + len(values)] = values

    def download_device(self, buf, *_):
        return buf.values

    def free_device(self, buf):
        pass

    def fixed_choose_device(self, logits, rows, vocab, choices, *, out, **lists):
        self.choices.append((choices.copy(), {k: v.values.copy() if isinstance(v, Buffer) else v for k, v in lists.items()}))
        out.values[0] = (logits.values[0] + 1) % vocab


class Decoder(forward.FixedDecoder):
    """Steps keep their tokens."""

    def __init__(self, slots=2, rows=None, **kw):
        self.config = c = forward.FixedConfig(**{**SIZES, **kw})
        self.backend, self.slots, self.rows = Library(), slots, rows or slots * c.positions
        self.lengths, self.prefix, self.steps = [0] * slots, None, []
        self._history, self._next = Buffer(np.zeros(c.positions + 1, np.int32)), Buffer(np.zeros(1, np.int32))
        self._allowed = Buffer(np.zeros((c.vocab + 31) // 32, np.uint32))

    def step_device(self, prompts, slots):
        prompts = [self._prompt(p) for p in prompts]
        if not all(len(p) for p in prompts) or sum(map(len, prompts)) > self.rows:
            raise InvalidInput("a step takes one non-empty prompt for each of its slots, within the decoder's rows")
        for p, s in zip(prompts, slots):
            self.steps.append((s, p.tolist()))
            self.lengths[s] += len(p)
        return Buffer([int(p[-1]) for p in prompts])


@pytest.mark.parametrize("prompt", [[3, 1, 4], (3, 1, 4), np.array([3, 1, 4], np.uint8), iter([3, 1, 4]),
                                    (t for t in (3, 1, 4)), dict.fromkeys([3, 1, 4]), map(int, "314")])
def test_generate_takes_tokens_from_any_iterable(prompt):
    model = Decoder()
    assert model.generate(prompt, 3, slot=1) == [5, 6, 7]
    assert model.steps == [(1, [3, 1, 4]), (1, [5]), (1, [6])]


def test_generate_takes_a_set_and_a_range():
    model = Decoder()
    assert model.generate({7}, 1) == [8] and model.generate(range(2, 5), 2, slot=1) == [5, 6]


@pytest.mark.parametrize("prompt", [5, None, "314", [1.5], iter([1.5]), iter([]), iter([50]), (t for t in (1, -1)),
                                    iter([[1, 2]]), np.array([[1, 2]]), np.array(3)])
def test_generate_refuses_what_gives_no_tokens(prompt):
    model = Decoder()
    with pytest.raises(InvalidInput):
        model.generate(prompt, 3)
    assert model.steps == [] and model.lengths == [0, 0]


@pytest.mark.parametrize("act,weight", [(10, 13), (10, 2), (3, 0), (13, 46), (14, 46), (15, 46), (15, 44)])
def test_biases_at_every_binary_point_of_the_logits(act, weight):
    """What reaches the operator is the bias at the logits' binary point, to half a step of 2^-13 or of a logit, or of
    2^-15 where the operator's shift, at most 46, asks for more bits."""
    model = Decoder(act_bits=act, weight_bits=weight, gain_bits=max(act, 12))
    bias = {4: 2.5, 7: -3.3, 9: 100.0, 11: 1e-5}
    model.generate([1], 2, bias=bias)
    for _, lists in model.backend.choices:
        assert 0 <= lists["bias_shift"] <= 46
        got = dict(zip(lists["bias_tokens"].tolist(), lists["bias_values"].astype(object) << lists["bias_shift"]))
        assert got.keys() == bias.keys()
        for t, v in bias.items():
            assert abs(got[t] / 2.0 ** (act + weight) - v) <= 2.0 ** (-1 - min(13, act + weight))


@pytest.mark.parametrize("act,weight,most", [(10, 13, 1 << 18), (15, 46, 1 << 16)])
def test_the_largest_biases(act, weight, most):
    model = Decoder(act_bits=act, weight_bits=weight, gain_bits=max(act, 12))
    model.generate([1], 1, bias={0: most - 2.0, 1: 2.0 - most})
    with pytest.raises(InvalidInput):
        model.generate([1], 1, bias={0: float(most)})


@pytest.mark.parametrize("token", [1.5, np.float32(2.25), "1", None, 50, -1, (1,), np.float64("nan"), 2 + 0j])
def test_biases_of_what_is_no_token_are_refused(token):
    """A fraction would turn into another token."""
    model = Decoder()
    with pytest.raises(InvalidInput):
        model.generate([1], 1, bias={0: 1.0, token: 2.0})
    assert model.steps == [] and model.generate([1], 1, bias={0: 1.0, np.int64(2): 2.0, np.uint8(3): 1, 4.0: 2}) == [2]
    assert model.backend.choices[-1][1]["bias_tokens"].tolist() == [0, 2, 3, 4]


@pytest.mark.parametrize("rows,pieces", [(None, [9]), (9, [9]), (8, [8, 1]), (4, [4, 4, 1]), (1, [1] * 9)])
def test_a_prefix_longer_than_a_step_is_shared(rows, pieces):
    model = Decoder(rows=rows)
    model.share(range(10, 19), 1)
    assert model.prefix == (1, 9) and model.lengths == [0, 9]
    assert [len(p) for _, p in model.steps] == pieces and {s for s, _ in model.steps} == {1}
    assert sum((p for _, p in model.steps), []) == list(range(10, 19))


def test_a_prefix_that_cannot_be_shared_leaves_no_tokens():
    for prompt, slot in (([], 0), ([1] * 25, 0), ([1, 50], 0), ([1], 2), ([1], -1), ([1] * 5 + [1.5], 0)):
        model = Decoder(rows=2)
        with pytest.raises(InvalidInput):
            model.share(prompt, slot)
        assert model.steps == [] and model.lengths == [0, 0] and model.prefix is None
    model = Decoder(rows=2)
    step = model.step_device

    def fails_later(prompts, slots):
        if model.steps:
            raise RuntimeError
        return step(prompts, slots)

    model.step_device = fails_later
    with pytest.raises(RuntimeError):
        model.share([1, 2, 3], 0)
    assert model.lengths == [0, 0] and model.prefix is None
