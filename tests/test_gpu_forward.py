"""The decoder over resident tensors: against the operators' definitions chained
on the host, the same trace for every batching, and the tensors committed."""
import fixed_reference as ref
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def model_tensors(config, seed):
    g = np.random.Generator(np.random.PCG64(seed))
    out = {}
    for name, shape in config.shapes().items():
        if name.endswith("gain"):
            t = (1 << config.gain_bits) + g.normal(0, 300, shape)
        elif name.endswith("bias"):
            t = g.normal(0, 200, shape)
        elif name == "wpe":
            t = g.normal(0, 100, shape)
        else:
            t = g.normal(0, (1 << config.weight_bits) * (1.0 if name == "wte" else 1.2 / np.sqrt(shape[0])), shape)
        out[name] = np.clip(np.rint(t), -32768, 32767).astype(np.int16)
    return out


def host_logits(config, t, tokens):
    """Logits after every token of one sequence."""
    from volta_mi355x import forward
    c = config
    act, exp = forward.activation_table(c.act_bits), forward.exponential_table(c)

    def linear(name, x, **kw):
        return ref.linear(x, t[name], bias=t[name + ".bias"], bias_shift=c.act_bits, shift=c.weight_bits, **kw)

    def norm(name, x, residual=None):
        return ref.norm(x, t[name + ".gain"], c.gain_bits - c.act_bits, c.norm_eps, bias=t[name + ".bias"],
                        residual=residual)

    n = len(tokens)
    h = ref.embed(tokens, t["wte"], shift=c.weight_bits - c.act_bits, positions=np.arange(n), position_table=t["wpe"])
    for i in range(c.layers):
        qkv = linear(f"h{i}.qkv", norm(f"h{i}.norm1", h)[0])
        q, k, v = np.split(qkv, [c.width, c.width + c.kv_width], axis=1)
        att = ref.attention(q.reshape(n, c.heads, c.dim), k.reshape(n, c.kv_heads, c.dim),
                            v.reshape(n, c.kv_heads, c.dim), exp, c.score_shift, True).reshape(n, c.width)
        y, h = norm(f"h{i}.norm2", linear(f"h{i}.proj", att), residual=h)
        h = linear(f"h{i}.down", linear(f"h{i}.up", y, table=act), residual=h)
    return ref.linear(norm("norm", h)[0], t["wte"].T, raw=True)


def configs():
    from volta_mi355x import forward
    return [forward.FixedConfig(layers=2, heads=4, kv_heads=4, dim=16, hidden=256, vocab=301, positions=96),
            forward.FixedConfig(layers=2, heads=6, kv_heads=2, dim=40, hidden=500, vocab=97, positions=200)]


@pytest.mark.parametrize("which", [0, 1])
def test_decoder_equals_the_operators_definitions(backend, which):
    from volta_mi355x import forward
    c = configs()[which]
    t = model_tensors(c, 3 + which)
    g = np.random.Generator(np.random.PCG64(8))
    seqs = [g.integers(0, c.vocab, n) for n in (70, 1, 33)]
    want = [host_logits(c, t, s) for s in seqs]
    dev = {name: backend.upload_device(v.reshape(-1)) for name, v in t.items()}
    model = forward.FixedDecoder(backend, c, dev, slots=3)
    try:
        # whole prompts, packed
        assert np.array_equal(model.step(seqs, [2, 0, 1]), np.stack([w[-1] for w in want]))
        # the same tokens one at a time, then in pieces
        for slot in range(3):
            model.reset(slot)
        for i, token in enumerate(seqs[0][:20]):
            assert np.array_equal(model.step([[token]], [1])[0], want[0][i]), i
        assert np.array_equal(model.step([seqs[0][20:50], seqs[2][:5]], [1, 0]), np.stack([want[0][49], want[2][4]]))
        assert np.array_equal(model.step([seqs[0][50:], seqs[2][5:6]], [1, 0]), np.stack([want[0][69], want[2][5]]))
        model.reset(0)
        first = model.generate(seqs[2], 4, slot=0)
        assert first[0] == int(np.argmax(want[2][-1]))
        model.reset(0)
        assert model.generate(seqs[2], 4, slot=0) == first
    finally:
        model.close()
        for b in dev.values():
            backend.free_device(b)


def test_decoder_refusals(backend):
    from volta_mi355x import InvalidInput, forward
    c = configs()[0]
    t = model_tensors(c, 1)
    dev = {name: backend.upload_device(v.reshape(-1)) for name, v in t.items()}
    with pytest.raises(InvalidInput):
        forward.FixedDecoder(backend, c, {k: v for k, v in dev.items() if k != "h1.up"})
    model = forward.FixedDecoder(backend, c, dev, slots=2)
    for prompts, slots in (([], []), ([[]], [0]), ([[1]], [2]), ([[1], [2]], [0, 0]), ([[1] * 97], [0]), ([[301]], [0]),
                           ([[-1]], [0])):
        with pytest.raises(InvalidInput):
            model.step(prompts, slots)
    assert model.lengths == [0, 0]
    assert model.step([[1, 2]], [1]).shape == (1, c.vocab) and model.lengths == [0, 2]
    model.close()
    for b in dev.values():
        backend.free_device(b)


@pytest.mark.parametrize("prompt", [np.array([1, (1 << 32) + 5]), np.array([(1 << 64) - 1], np.uint64), [1.5],
                                    [[1, 2], [3, 4]], [1 << 40], ["7"]])
def test_decoder_refuses_prompts_that_are_no_row_of_tokens(backend, prompt):
    """Tokens that an i32 would hold as another one, fractions, and prompts of more than one dimension."""
    from volta_mi355x import InvalidInput, forward
    c = configs()[0]
    dev = {name: backend.upload_device(v.reshape(-1)) for name, v in model_tensors(c, 1).items()}
    model = forward.FixedDecoder(backend, c, dev, slots=2)
    try:
        with pytest.raises(InvalidInput):
            model.step([prompt, [3]], [0, 1])
        assert model.lengths == [0, 0]
        same = [model.step([p], [0]) for p in (np.array([3, 5], np.uint8), [3, 5]) if model.reset(0) is None]
        assert np.array_equal(*same)
    finally:
        model.close()
        for b in dev.values():
            backend.free_device(b)


def scale_configs():
    from volta_mi355x import forward
    sizes = dict(layers=1, heads=4, kv_heads=2, dim=16, hidden=32, vocab=50, positions=24)
    return [forward.FixedConfig(**sizes), forward.FixedConfig(**sizes, act_bits=12, weight_bits=9, gain_bits=13)]


@pytest.mark.parametrize("which", [0, 1])
def test_decoder_of_quantised_tensors_is_near_the_real_model(backend, which):
    """Real tensors quantised at the binary points that the config states, in a model whose block adds its two biases
    only (proj and down are zero), against the real model in 64-bit floating point.

    The bound, with u and w half a step of activations and of weights: an element of the stream is off by w (wte), 2 u
    (its rounding, and wpe) and 2 (w + u) (each bias and its rounding), D in all.  Centred, by at most 2 D; the deviation
    by D and the roundings of eps and of the root.  The normalised value's quotient, gain and bias add theirs, and the
    product with wte its own w.  Values stay inside 16 bits (asserted), so nothing is clamped."""
    from volta_mi355x import forward
    c = scale_configs()[which]
    g = np.random.Generator(np.random.PCG64(which))
    real = {}
    for name, shape in c.shapes().items():
        spread = 0.0 if name in ("h0.proj", "h0.down") else 0.4 if name.endswith("bias") else 0.6
        real[name] = (1.0 + 0.2 * g.uniform(-1, 1, shape)) if name.endswith("gain") else spread * g.uniform(-1, 1, shape)
    tokens = g.integers(0, c.vocab, c.positions)

    def logits(t):
        h = t["wte"][tokens] + t["wpe"] + t["h0.proj.bias"] + t["h0.down.bias"]
        centred = h - h.mean(1, keepdims=True)
        spread = np.sqrt((centred ** 2).mean(1, keepdims=True) + c.eps)
        y = centred / spread * t["norm.gain"] + t["norm.bias"]
        return y @ t["wte"].T, centred / spread, spread, y

    want, hat, spread, y = logits(real)
    u, w, n = 2.0 ** -(c.act_bits + 1), 2.0 ** -(c.weight_bits + 1), c.width
    d = (w + 2 * u) + 2 * (w + u)
    off = d + 1 / (n << c.act_bits) + 0.25 / (n ** 2 * 4 ** c.act_bits * spread)
    d_hat = (2 * d + np.abs(hat) * off) / (spread - off)
    d_y = d_hat * real["norm.gain"] + (np.abs(hat) + d_hat) * 2.0 ** -(c.gain_bits + 1) + 2 * u
    bound = d_y @ (np.abs(real["wte"]) + w).T + np.abs(y).sum(1, keepdims=True) * w
    assert np.abs(y).max() + d_y.max() < 2.0 ** (15 - c.act_bits)

    dev = {}
    for name, t in real.items():
        q = np.rint(t * 2.0 ** c.bits(name))
        assert np.abs(q).max() < 32768
        dev[name] = backend.upload_device(q.astype(np.int16).reshape(-1))
    model = forward.FixedDecoder(backend, c, dev)
    try:
        got = np.concatenate([model.step([[int(t)]], [0]) for t in tokens]) / 2.0 ** (c.act_bits + c.weight_bits)
    finally:
        model.close()
        for b in dev.values():
            backend.free_device(b)
    assert (np.abs(got - want) <= bound).all()
    # the bound tells a tensor at twice its scale
    for name in ("wte", "wpe", "h0.proj.bias", "h0.down.bias", "norm.gain", "norm.bias"):
        assert (np.abs(logits({**real, name: 2 * real[name]})[0] - want) > 2 * bound).any(), name


def test_the_same_tensors_run_and_are_committed(backend, oracle):
    """One layer's matrices: placed and committed from the resident buffers that the decoder runs."""
    from volta_mi355x import forward, ligero, workloads
    c = forward.FixedConfig(layers=1, heads=4, kv_heads=4, dim=16, hidden=256, vocab=64, positions=32)
    t = model_tensors(c, 5)
    dev = {name: backend.upload_device(v.reshape(-1)) for name, v in t.items()}
    slots, total = workloads.block_layout([(n, *c.shapes()[f"h0.{n}"]) for n in ("qkv", "proj", "up", "down")])
    params = ligero.LigeroParams(total >> 8, 8, 32, 10, 0)
    placements = [ligero.ResidentWeightPlacement(dev[f"h0.{s.name}"], 0, s.k, s.n, s.offset, s.stride, total)
                  for s in slots]
    model = forward.FixedDecoder(backend, c, dev)
    before = model.step([[1, 2, 3]], [0])
    root, matrix = ligero.commit_resident_from_device(backend, placements, params, bytes(range(32)))
    model.reset(0)
    assert np.array_equal(model.step([[1, 2, 3]], [0]), before)
    assert np.array_equal(before[0], host_logits(c, t, [1, 2, 3])[-1])
    packed = backend.download_device(matrix.weights)
    for s in slots:
        block = np.lib.stride_tricks.as_strided(packed[s.offset:], (s.k, s.n), (2 * s.stride, 2))
        assert np.array_equal(block, t[f"h0.{s.name}"])
    assert len(root) == 32
    model.close()
    for b in (matrix.weights, matrix.pads, matrix.encoded, matrix.tree.storage, *dev.values()):
        backend.free_device(b)
