"""The decoder with head norms, rotary positions, a window, a shared prefix and a choice under penalties, against the
operators' definitions chained on the host."""
import fixed_reference as ref
import numpy as np
import pytest
import serving_reference as want
from test_gpu_forward import model_tensors

pytestmark = pytest.mark.gpu


def host_logits(config, t, tokens):
    """Logits after every token of one sequence."""
    from volta_mi355x import forward
    c = config
    act, exp, angles = forward.activation_table(c.act_bits), forward.exponential_table(c), forward.rotation_table(c)

    def linear(name, x, **kw):
        return ref.linear(x, t[name], bias=t[name + ".bias"], bias_shift=c.act_bits, shift=c.weight_bits, **kw)

    def norm(name, x, residual=None):
        return ref.norm(x, t[name + ".gain"], c.gain_bits - c.act_bits, c.norm_eps, bias=t[name + ".bias"],
                        residual=residual)

    n = len(tokens)
    seen = want.window_seen(n, n, c.window or n, c.sinks)
    learned = {} if c.rotary else dict(positions=np.arange(n), position_table=t["wpe"])
    h = ref.embed(tokens, t["wte"], shift=c.weight_bits - c.act_bits, **learned)
    for i in range(c.layers):
        qkv = linear(f"h{i}.qkv", norm(f"h{i}.norm1", h)[0])
        qk, v = np.split(qkv, [c.width + c.kv_width], axis=1)
        kw = dict(q_gain=t[f"h{i}.q_norm.gain"], k_gain=t[f"h{i}.k_norm.gain"]) if c.head_norm else {}
        qk = want.rotate(qk, c.heads, c.dim, gain_shift=c.gain_bits - c.act_bits, eps=c.head_eps, angles=angles,
                         positions=np.arange(n), rotated=c.rotary, adjacent=c.adjacent, **kw)
        q, k = np.split(qk, [c.width], axis=1)
        att = want.attention(q.reshape(n, c.heads, c.dim), k.reshape(n, c.kv_heads, c.dim), v.reshape(n, c.kv_heads, c.dim),
                             seen, exp, c.score_shift).reshape(n, c.width)
        y, h = norm(f"h{i}.norm2", linear(f"h{i}.proj", att), residual=h)
        h = linear(f"h{i}.down", linear(f"h{i}.up", y, table=act), residual=h)
    return ref.linear(norm("norm", h)[0], t["wte"].T, raw=True)


BASE = dict(layers=2, heads=4, kv_heads=2, dim=16, hidden=200, vocab=301, positions=120)


@pytest.fixture
def decoder(backend):
    """Makes a decoder and its tensors from a configuration."""
    from volta_mi355x import forward
    open_models, held = [], []

    def make(slots=3, seed=4, **kw):
        c = forward.FixedConfig(**{**BASE, **kw})
        t = model_tensors(c, seed)
        dev = {name: backend.upload_device(v.reshape(-1)) for name, v in t.items()}
        held.extend(dev.values())
        open_models.append(forward.FixedDecoder(backend, c, dev, slots=slots))
        return open_models[-1], c, t

    yield make
    for m in open_models:
        m.close()
    for b in held:
        backend.free_device(b)


VARIANTS = [dict(rotary=16), dict(rotary=16, adjacent=True, head_norm=True), dict(rotary=10, head_norm=True, window=20),
            dict(head_norm=True), dict(window=30, sinks=3), dict(rotary=8, window=1, sinks=1, kv_heads=4),
            dict(rotary=40, dim=40, heads=6, window=64, sinks=70, head_norm=True), dict(rotary=16, window=500)]


@pytest.mark.parametrize("kw", VARIANTS)
def test_decoder_variants_equal_the_operators_definitions(decoder, kw):
    model, c, t = decoder(**kw)
    g = np.random.Generator(np.random.PCG64(8))
    seqs = [g.integers(0, c.vocab, n) for n in (100, 1, 33)]
    want_all = [host_logits(c, t, s) for s in seqs]
    assert np.array_equal(model.step(seqs, [2, 0, 1]), np.stack([w[-1] for w in want_all]))
    for slot in range(3):
        model.reset(slot)
    for i, token in enumerate(seqs[0][:25]):
        assert np.array_equal(model.step([[token]], [1])[0], want_all[0][i]), i
    assert np.array_equal(model.step([seqs[0][25:60], seqs[2][:5]], [1, 0]), np.stack([want_all[0][59], want_all[2][4]]))
    assert np.array_equal(model.step([seqs[0][60:], seqs[2][5:6]], [1, 0]), np.stack([want_all[0][99], want_all[2][5]]))


@pytest.mark.parametrize("kw", [{}, dict(rotary=16, head_norm=True)])
def test_a_shared_prefix_is_the_beginning_of_every_sequence(decoder, kw):
    from volta_mi355x import InvalidInput
    model, c, t = decoder(slots=4, **kw)
    g = np.random.Generator(np.random.PCG64(9))
    start = g.integers(0, c.vocab, 70)
    seqs = [g.integers(0, c.vocab, n) for n in (30, 1, 12)]
    want_all = [host_logits(c, t, np.concatenate([start, s])) for s in seqs]
    model.share(start, 1)
    assert np.array_equal(model.step(seqs, [0, 2, 3]), np.stack([w[-1] for w in want_all]))
    model.reset(0)
    for i, token in enumerate(seqs[0][:10]):
        assert np.array_equal(model.step([[token]], [0])[0], want_all[0][70 + i]), i
    for call in (lambda: model.step([[1]], [1]), lambda: model.reset(1), lambda: model.share(start, 2),
                 lambda: model.step([[1] * 41], [0]), lambda: model.generate([1], 51, slot=2)):
        with pytest.raises(InvalidInput):
            call()
    assert model.lengths == [10, 70, 1, 12]
    model.reset(2)
    first = model.generate(seqs[2], 6, slot=2)
    assert first[0] == int(np.argmax(want_all[2][-1]))
    model.unshare()
    assert np.array_equal(model.step([seqs[1]], [1])[0], host_logits(c, t, seqs[1])[-1])
    with pytest.raises(InvalidInput):
        model.share(start, 0)


def test_a_window_and_a_shared_prefix_are_refused(decoder):
    from volta_mi355x import InvalidInput
    model, c, _ = decoder(window=9)
    with pytest.raises(InvalidInput):
        model.share([1, 2], 0)
    assert model.lengths == [0, 0, 0] and model.prefix is None


@pytest.mark.parametrize("kw", [dict(), dict(repetition=1.3), dict(frequency=0.7, presence=0.25),
                                dict(repetition=0.8, bias={5: 3.0, 17: -1.5}), dict(bias={200: 1000.0})])
@pytest.mark.parametrize("masked", [False, True])
def test_generate_under_penalties_biases_and_masks(decoder, kw, masked):
    model, c, t = decoder(rotary=16, head_norm=True, window=25, sinks=2)
    g = np.random.Generator(np.random.PCG64(3))
    prompt = g.integers(0, c.vocab, 20)
    allowed = g.random(c.vocab) < 0.4 if masked else None
    unit = c.act_bits + c.weight_bits
    sequence, answer = list(prompt), []
    for _ in range(6):
        row = dict(history=sequence, mask=allowed, repetition=round(65536 * kw.get("repetition", 1.0)),
                   frequency=round(kw.get("frequency", 0.0) * 2 ** unit), presence=round(kw.get("presence", 0.0) * 2 ** unit),
                   biases=[(i, round(v * 2 ** 13)) for i, v in kw.get("bias", {}).items()])
        tokens, _ = want.choose(host_logits(c, t, np.array(sequence))[-1:], [row], bias_shift=unit - 13)
        answer.append(int(tokens[0]))
        sequence.append(answer[-1])
    assert model.generate(prompt, 6, allowed=allowed, **kw) == answer


def test_generate_with_a_grammar(decoder):
    """A function gives the mask for the answer so far; nothing allowed ends it."""
    model, c, t = decoder()
    seen = []

    def allowed(answer):
        seen.append(answer)
        mask = np.zeros(c.vocab, bool)
        if len(answer) < 3:
            mask[len(answer) * 100:len(answer) * 100 + 7] = True
        return mask

    answer = model.generate([1, 2, 3], 9, allowed=allowed)
    assert [a // 100 for a in answer] == [0, 1, 2] and all(a % 100 < 7 for a in answer)
    assert seen == [answer[:n] for n in range(4)]


def test_generate_refusals(decoder):
    from volta_mi355x import InvalidInput
    model, c, _ = decoder()
    nan = float("nan")
    for args, kw in ((([1], 1, 3), {}), (([1], 1, -1), {}), (([1], 121), {}), (([301], 1), {}), (([], 1), {}),
                     (([1], 1), dict(repetition=0.0)), (([1], 1), dict(repetition=-1.0)), (([1], 1), dict(repetition=nan)),
                     (([1], 1), dict(repetition=65536.0)), (([1], 1), dict(frequency=1e15)), (([1], 1), dict(presence=nan)),
                     (([1], 1), dict(bias={301: 1.0})), (([1], 1), dict(bias={-1: 1.0})), (([1], 1), dict(bias={1: 1e6})),
                     (([1], 1), dict(bias={1: nan})), (([1], 1), dict(allowed=np.ones(300, bool))),
                     (([1], 1), dict(allowed=np.ones(301))), (([1], 1), dict(allowed=lambda a: [True]))):
        with pytest.raises(InvalidInput):
            model.generate(*args, **kw)
    assert model.lengths == [0, 0, 0]
    assert model.generate([1], 0) == []
    assert len(model.generate([1], 120)) == 120 and model.lengths[0] == 120



@pytest.mark.parametrize("rows", [1, 7, 69, 70])
def test_a_prefix_longer_than_the_decoders_rows(backend, rows):
    """Shared in steps of those: the same logits behind it as behind the tokens themselves."""
    from volta_mi355x import forward
    c = forward.FixedConfig(**BASE, rotary=16)
    t = model_tensors(c, 4)
    g = np.random.Generator(np.random.PCG64(rows))
    start, seq = g.integers(0, c.vocab, 70), g.integers(0, c.vocab, 6)
    dev = {name: backend.upload_device(v.reshape(-1)) for name, v in t.items()}
    model = forward.FixedDecoder(backend, c, dev, slots=2, rows=rows)
    try:
        model.share(start, 0)
        want_all = host_logits(c, t, np.concatenate([start, seq]))
        for i, token in enumerate(seq):
            assert np.array_equal(model.step([[token]], [1])[0], want_all[70 + i]), i
    finally:
        model.close()
        for b in dev.values():
            backend.free_device(b)
