"""The serving operators' kernels, each by cases that reach it: which kernel a call takes is a rule on its sizes.

Behind a prefix the rule is the library's own (fixed_rules.hpp, built for the host too): the CPU tests hold every case
to the kernel it is for, so that a change of the rule shows here.  Without a prefix, and for the other operators,
the sizes are on both sides of the rules' bounds for 256 CUs."""
import ctypes
import pathlib

import fixed_reference as ref
import numpy as np
import pytest
import serving_reference as want
from test_gpu_fixed import exponentials, full, gen, normal
from test_gpu_serving import check_choose, check_prefix, check_window, choice_rows, make, run, run_rotate

LIB = pathlib.Path(__file__).resolve().parent.parent / "volta-zk_amd" / "libgl64_check.so"
ALL = (1 << 64) - 1


def prefix_limit(dim, kv_heads, heads, prefix, counts, lengths):
    """Sequences of up to so many rows read the prefix together."""
    lib = ctypes.CDLL(str(LIB))
    lib.glc_prefix_limit.restype = ctypes.c_size_t
    lib.glc_prefix_limit.argtypes = [ctypes.c_size_t] * 4 + [ctypes.c_void_p] * 2 + [ctypes.c_size_t]
    c, l = (np.ascontiguousarray(x, np.uint32) for x in (counts, lengths))
    return lib.glc_prefix_limit(dim, kv_heads, heads, prefix, c.ctypes.data, l.ctypes.data, len(c))


# ---- behind a prefix ------------------------------------------------------------------------------

def behind_prefix(q, k, v, pk, pv, table, shift, causal):
    """serving_reference.attention of every sequence behind the prefix, whose scores are taken for all rows at once; in
    whole numbers below 2^53, held in doubles."""
    heads, kv_heads = q[0].shape[1], pk.shape[1]
    e_of = np.minimum(table, 1 << 14).astype(np.float64)
    rows = np.concatenate(q).astype(np.float64)
    out = np.zeros(rows.shape, np.int16)
    for h in range(heads):
        g = h * kv_heads // heads
        z = np.floor(rows[:, h] @ pk[:, g].astype(np.float64).T / 2.0 ** shift)
        own, row = [], 0
        for i, part in enumerate(q):
            n, tokens = len(part), len(k[i])
            zo = np.floor(rows[row:row + n, h] @ k[i][:, g].astype(np.float64).T / 2.0 ** shift)
            if causal:
                zo[np.arange(tokens)[None] > (tokens - n + np.arange(n))[:, None]] = -np.inf
            own.append(zo)
            row += n
        top = np.maximum(z.max(1), np.concatenate([o.max(1, initial=-np.inf) for o in own]))
        e = e_of[np.minimum(top[:, None] - z, len(table) - 1).astype(np.int64)]
        sums, total, row = e @ pv[:, g].astype(np.float64), e.sum(1), 0
        for i, zo in enumerate(own):
            at = slice(row, row + len(zo))
            eo = np.where(zo == -np.inf, 0, e_of[np.minimum(top[at, None] - zo, len(table) - 1).astype(np.int64)])
            sums[at] += eo @ v[i][:, g].astype(np.float64)
            total[at] += eo.sum(1)
            row += len(zo)
        s, t = sums.astype(np.int64), total.astype(np.int64)[:, None]
        out[:, h] = np.where(t > 0, np.floor_divide(2 * s + t, np.maximum(2 * t, 1)), 0)
    return np.split(out, np.cumsum([len(p) for p in q])[:-1])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim,ends", [(5, False), (64, True), (128, True)])
def test_reference_of_all_sequences(causal, dim, ends):
    counts, lengths = [3, 0, 1, 9], [7, 5, 1, 40] if causal else [7, 5, 0, 4]
    q, k, v, pk, pv = make(dim, counts, lengths, 4, 2, dim, 90, ends)
    for shift in (8, 13, 24):
        got = behind_prefix(q, k, v, pk, pv, exponentials(), shift, causal)
        for i, (n, t) in enumerate(zip(counts, lengths)):
            assert np.array_equal(got[i], want.attention(q[i], np.concatenate([pk, k[i]]), np.concatenate([pv, v[i]]),
                                                         want.prefix_seen(n, 90, t, causal), exponentials(), shift))


class Case:
    """A call behind a prefix: its sequences, and which of them are to read the prefix together."""

    def __init__(self, together, dim, kv_heads, heads, prefix, counts, lengths, **kw):
        self.together, self.sizes, self.counts, self.lengths, self.kw = together, (dim, kv_heads, heads, prefix), counts, lengths, kw

    def took(self):
        """The outcome for its sequences: none, some or all together."""
        limit = prefix_limit(*self.sizes, self.counts, self.lengths)
        rows = [n * (self.sizes[2] // self.sizes[1]) for n in self.counts if n]
        return {0: "none", len(rows): "all"}.get(sum(r <= limit for r in rows), "some")

    def check(self, b, seed):
        dim, kv_heads, heads, prefix = self.sizes
        kw = dict(self.kw)
        causal, ends = kw.pop("causal", True), kw.pop("ends", False)
        shift = kw.pop("shift", None) or max(8, round(np.log2(np.sqrt(dim) * 1e6 / 1280.0)))
        q, k, v, pk, pv = make(seed, self.counts, self.lengths, heads, kv_heads, dim, prefix, ends)
        got = run(b, q, k, v, pk, pv, shift, exponentials(), causal=causal, **kw)
        expect = behind_prefix(q, k, v, pk, pv, exponentials(), shift, causal)
        for i, (x, y) in enumerate(zip(got, expect)):
            assert np.array_equal(x, y), (i, self.counts[i], self.lengths[i])

    def __repr__(self):
        return f"{self.together}-{'x'.join(map(str, self.sizes))}-{len(self.counts)}x{max(self.counts)}"


def short(seed, n, longest, least=1):
    return [int(x) for x in gen(seed).integers(least, longest + 1, n)]


TOKENS = [Case("all", dim, 4, heads, prefix, [1] * 31, short(dim + heads, 31, 200))
          for dim in (1, 33, 64, 65, 96, 128) for heads in (4, 12, 32) for prefix in (8129, 8191, 8192)]
BATCHES = [Case("all", dim, 8, 16, 8192, [1] * batch, short(batch, batch, 90))
           for dim in (64, 128) for batch in (2, 8, 63, 64, 65, 128, 130, 192) if batch > 2 or dim == 64]
ENDS = [Case("all", dim, 4, 8, 4100, [1] * 40, short(dim, 40, 100), shift=shift, ends=True)
        for dim in (64, 128) for shift in (8, 13, 17, 24)]
APART = []
for _dim in (40, 64, 96, 128):
    for _causal in (True, False):
        _counts = [int(n) for n in gen(_dim).integers(0, 4, 70)]
        _lengths = [max(n, m) if _causal else m for n, m in zip(_counts, short(_dim, 70, 300, 0))]
        _order = [int(i) for i in gen(_dim + 1).permutation(70)]
        APART.append(Case("all", _dim, 4, 12, 8192, _counts, _lengths, causal=_causal, row_gap=2, gap=3, offset=1, order=_order))
        APART.append(Case("all", _dim, 8, 8, 8192, [2] * 66, [n + 2 for n in _lengths[:66]], causal=_causal, row_gap=1))
PROMPTS_TOGETHER = [Case("all", dim, 4, heads, prefix, [1] * 8 + [200, 1, 130] + [1] * 8, [90] * 8 + [230, 1, 130] + [70] * 8)
                    for dim in (64, 128) for heads in (4, 8) for prefix in (2200, 4099)]
PROMPTS_TOGETHER += [Case("all", 64, 4, 4, 4100, [100] * 20, [100] * 20), Case("all", 128, 4, 4, 4100, [100] * 20, [120] * 20)]
SOME = [Case("some", 64, 4, 8, 4100, [1] * 16 + [200] * 10 + [1] * 15, [90] * 16 + [230] * 10 + [1] * 15, row_gap=1),
        Case("some", 40, 8, 8, 3000, [200] * 10 + [1, 3] * 15, [200] * 10 + [60, 3] * 15, causal=False),
        Case("some", 128, 4, 8, 4100, [200] * 5 + [1] * 64 + [200] * 5, [230] * 5 + [90] * 64 + [230] * 5, row_gap=1),
        Case("some", 128, 8, 8, 4100, [200] * 5 + [1] * 64 + [200] * 5, [230] * 5 + [90] * 64 + [230] * 5,
             order=[int(i) for i in gen(3).permutation(74)])]
# prompts: two teams up to a workgroup a CU, one above; tokens: scores kept in registers, in LDS, and in memory
NONE = [Case("none", dim, kv, heads, 300, [100] * n, [n + 100 for n in short(dim, n, 50)])
        for dim in (64, 96, 128) for kv, heads, n in ((3, 6, 3), (8, 16, 20), (4, 4, 100))]
NONE += [Case("none", dim, 4, 8, prefix, [1, 2, 1], [1, 40, 64])
         for dim in (64, 128) for prefix in (100, 350, 600, 1000, 2000)]
PREFIXES = TOKENS + BATCHES + ENDS + APART + PROMPTS_TOGETHER + SOME + NONE


@pytest.mark.parametrize("case", PREFIXES, ids=repr)
def test_prefix_cases_take_the_kernel_that_they_are_for(case):
    assert case.took() == case.together


@pytest.mark.gpu
@pytest.mark.parametrize("case", PREFIXES, ids=repr)
def test_prefix(backend, case):
    assert case.took() == case.together
    case.check(backend, case.sizes[0] + len(case.counts))


# ---- over a window --------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dim", [40, 64, 65, 128])
@pytest.mark.parametrize("window,sinks", [(64, 0), (449, 64), (512, 1), (600, 70), (700, 0), (961, 64), (1500, 3)])
@pytest.mark.parametrize("batch,heads,kv_heads", [(1, 1, 1), (3, 8, 2), (80, 4, 4)])
def test_window_of_tokens(backend, dim, window, sinks, batch, heads, kv_heads):
    """Tiles of a window on both sides of what a workgroup keeps in registers (8 for heads over 64, 16), in LDS, and of
    what it reads alone."""
    lengths = [2000] + short(batch + window, batch - 1, 1900)
    check_window(backend, window, [1] * batch, lengths, heads, kv_heads, dim, window, sinks, row_gap=batch == 3)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [40, 64, 96, 128])
@pytest.mark.parametrize("length,heads,kv_heads", [(1100, 4, 2), (600, 60, 60), (2200, 16, 16)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (64, 64), (500, 70)])
def test_window_of_prompts(backend, dim, length, heads, kv_heads, window, sinks):
    """Two teams up to a workgroup a CU, one above (60 key heads of 600 tokens: 300; 16 of 2,200: 288)."""
    check_window(backend, dim + length, [length], [length], heads, kv_heads, dim, window, sinks)


# ---- heads normed and rotated, two heads a lane ---------------------------------------------------

def rotate_many(x, heads, dim, *, q_gain=None, k_gain=None, gain_shift=0, eps=1, angles=None, positions=None, rotated=0,
                adjacent=False, angle_shift=14):
    """serving_reference.rotate for many rows at once: roots from doubles, put right in whole numbers."""
    h = x.astype(np.int64).reshape(len(x), -1, dim)
    for at, gain in ((slice(0, heads), q_gain), (slice(heads, None), k_gain)):
        if gain is None:
            continue
        v = dim * (h[:, at] ** 2).sum(-1, keepdims=True) + eps
        root = np.sqrt(v.astype(np.float64)).astype(np.int64)
        root -= root * root > v
        root += (root + 1) * (root + 1) <= v
        below = root << gain_shift
        h[:, at] = ref.sat(np.floor_divide(2 * dim * h[:, at] * gain.astype(np.int64) + below, 2 * below))
    if rotated:
        inside = (positions >= 0) & (positions < len(angles))
        c, s = np.moveaxis(angles.astype(np.int64)[np.where(inside, positions, 0)], -1, 0)[:, :, None]  # rows x 1 x pairs
        pairs = rotated // 2
        one = slice(0, rotated, 2) if adjacent else slice(0, pairs)
        two = slice(1, rotated, 2) if adjacent else slice(pairs, rotated)
        a, b, turned = h[inside][..., one], h[inside][..., two], h[inside].copy()
        c, s = c[inside], s[inside]
        turned[..., one] = ref.sat(ref.rs(a * c - b * s, angle_shift))
        turned[..., two] = ref.sat(ref.rs(a * s + b * c, angle_shift))
        h[inside] = turned
    return h.reshape(x.shape).astype(np.int16)


def rotate_inputs(seed, rows, heads, kv_heads, dim, rotated, *, gains="qk", ends=False, adjacent=False, gain_shift=2, eps=1,
                  places=50):
    g = gen(seed)
    one = (lambda shape, std: full(g, shape)) if ends else (lambda shape, std: normal(g, shape, std))
    x = one((rows, (heads + kv_heads) * dim), 1500)
    x[g.random(rows) < 0.1] = 0
    args = dict(gain_shift=gain_shift, eps=eps, adjacent=adjacent, rotated=rotated)
    for name in gains:
        args[f"{name}_gain"] = one(dim, 4000)
    if rotated:
        args.update(angles=one((places, rotated // 2, 2), 9000), positions=g.integers(-2, places + 2, rows).astype(np.int32))
    return x, args


@pytest.mark.parametrize("dim,rotated", [(1, 0), (7, 4), (32, 32), (64, 40), (128, 128)])
@pytest.mark.parametrize("gains", ["", "q", "k", "qk"])
@pytest.mark.parametrize("adjacent,ends", [(False, False), (True, True)])
def test_reference_of_many_rows(dim, rotated, gains, adjacent, ends):
    for gain_shift, eps in ((0, 1), (15, 1 << 40), (2, 77)):
        x, args = rotate_inputs(dim, 40, 3, 2, dim, rotated, gains=gains, ends=ends, adjacent=adjacent, gain_shift=gain_shift,
                                eps=eps)
        assert np.array_equal(rotate_many(x, 3, dim, **args), want.rotate(x, 3, dim, **args))


# heads of a launch from which a lane takes two, for 256 CUs and 4, 8 and 16 lanes a head
TWO_HEADS = {32: 131072, 64: 65536, 128: 32768}


@pytest.mark.gpu
@pytest.mark.parametrize("dim,rotated", [(1, 0), (24, 24), (31, 18), (32, 32), (33, 10), (64, 64), (64, 22), (80, 80), (127, 126),
                                         (128, 128)])
@pytest.mark.parametrize("less", [1, 0, -1])
def test_two_heads_a_lane(backend, dim, rotated, less):
    """One head a row, from one below to one above the number of heads: the last group is whole or not."""
    heads = TWO_HEADS[32 if dim <= 32 else 64 if dim <= 64 else 128] - less
    for adjacent in (False, True):
        x, args = rotate_inputs(dim + less, heads, 1, 0, dim, rotated, gains="q", adjacent=adjacent)
        assert np.array_equal(run_rotate(backend, x, 1, 0, dim, **args), rotate_many(x, 1, dim, **args))


@pytest.mark.gpu
@pytest.mark.parametrize("dim,rotated", [(20, 16), (32, 32), (48, 48), (64, 64), (64, 30), (65, 64), (128, 96), (128, 128)])
@pytest.mark.parametrize("gains", ["q", "k", "qk"])
@pytest.mark.parametrize("in_place", [False, True])
def test_two_heads_a_lane_of_rows(backend, dim, rotated, gains, in_place):
    """Rows of 4 + 3 heads, of which one kind or both are normed; strides, and an output in place."""
    rows = TWO_HEADS[32 if dim <= 32 else 64 if dim <= 64 else 128] // 7 + 3
    x, args = rotate_inputs(dim, rows, 4, 3, dim, rotated, gains=gains, adjacent=rotated % 4 == 0, gain_shift=3, eps=4096)
    got = run_rotate(backend, x, 4, 3, dim, in_place=in_place, x_gap=5, out_gap=2, offset=3, **args)
    assert np.array_equal(got, rotate_many(x, 4, dim, **args))


@pytest.mark.gpu
@pytest.mark.parametrize("dim,rotated", [(32, 32), (64, 64), (128, 128)])
@pytest.mark.parametrize("gain_shift,eps", [(0, 1), (15, 1 << 40), (3, 7)])
def test_two_heads_a_lane_of_values_at_the_ends(backend, dim, rotated, gain_shift, eps):
    x, args = rotate_inputs(dim, TWO_HEADS[dim] // 5 + 1, 3, 2, dim, rotated, ends=True, gain_shift=gain_shift, eps=eps)
    assert np.array_equal(run_rotate(backend, x, 3, 2, dim, **args), rotate_many(x, 3, dim, **args))


# ---- where no workspace may grow ------------------------------------------------------------------

class Scope:
    """A backend whose calls of one operator run in a coarse timing scope, in which no workspace may be allocated."""

    def __init__(self, b, operator):
        self.b, self.operator, self.calls = b, operator, 0

    def __getattr__(self, name):
        f = getattr(self.b, name)
        if name != self.operator:
            return f

        def call(*args, **kw):
            live = self.b.get_stats()["live_device_bytes"]
            assert self.b.lib.volta_cuda_begin_coarse_timing(self.b.raw, 0) == 0
            result = f(*args, **kw)
            assert self.b.lib.volta_cuda_end_coarse_timing(self.b.raw) == 0
            assert self.b.get_stats()["live_device_bytes"] == live
            self.calls += 1
            return result

        return call


@pytest.fixture
def scope():
    """Makes a context of its own, without any workspace yet, in such a scope."""
    from volta_mi355x import Backend
    made = []

    def make_scope(operator):
        made.append((Backend(timing_policy=1), operator))
        return Scope(*made[-1])

    yield make_scope
    for b, _ in made:
        b.close()


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 31, 2047, 2048, 2049, 4096, 6000])
@pytest.mark.parametrize("adjusted", ["new", "in place", None])
@pytest.mark.parametrize("rows", [3, 70, 130])
def test_choose_without_a_workspace(scope, vocab, adjusted, rows):
    """A workgroup a row, with a count and a sum for each token of 2,048 at a time."""
    b = scope("fixed_choose_device")
    g = gen(vocab + rows)
    logits = np.rint(g.normal(0, 3000, (rows, vocab))).astype(np.int64)
    some = choice_rows(g, rows, vocab, history=60, biases=11)
    some[0]["history"] = np.concatenate([np.full(33000, vocab // 2), g.integers(-3, vocab + 3, 500)])
    some[-1]["biases"] = [(int(t), int(v)) for t, v in zip(g.integers(-3, vocab + 3, 700), g.integers(-9999, 9999, 700))]
    check_choose(b, logits, some, bias_shift=5, adjusted=adjusted, gap=3, offset=1, mask_gap=1, junk=2)
    assert b.calls == 1


@pytest.mark.gpu
def test_choose_without_a_workspace_at_the_ends(scope):
    b = scope("fixed_choose_device")
    g = gen(9)
    logits = g.choice(np.array([-(1 << 63), -(1 << 63) + 1, (1 << 63) - 1, 1 << 62, 1 << 35, -(1 << 35), -1, 0, 1], np.int64),
                      (66, 2300))
    some = choice_rows(g, 66, 2300, history=900, biases=50)
    for i, r in enumerate(some):
        r["frequency"] = ((1 << 63) - 1, -(1 << 63), 1 << 40, 1 << 31, (1 << 31) - 1, 5)[i % 6]
        r["presence"] = -r["frequency"] - 1
        r["biases"] = [(t, int(g.choice([-(1 << 31), (1 << 31) - 1, 1]))) for t, _ in r["biases"]]
    check_choose(b, logits, some, bias_shift=46)
    check_choose(b, np.full((66, 2300), -(1 << 63)), [dict(some[0], mask=np.zeros(2300, bool))] * 66, bias_shift=46)


@pytest.mark.gpu
@pytest.mark.parametrize("case", [BATCHES[-1], SOME[0], SOME[2], PROMPTS_TOGETHER[0], PROMPTS_TOGETHER[-1], APART[0]], ids=repr)
def test_prefix_without_a_workspace(scope, case):
    """Each sequence by itself, its scores computed twice."""
    b = scope("fixed_attention_device")
    assert case.took() == case.together
    case.check(b, 5)
    assert b.calls == 1


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1500, 3), (2500, 100)])
def test_window_without_a_workspace(scope, dim, window, sinks):
    b = scope("fixed_attention_device")
    check_window(b, dim, [1, 3, 1], [3000, 2900, 700], 8, 4, dim, window, sinks)
    assert b.calls == 1


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_workspaces_that_grow_between_calls(dim):
    """Small calls before large ones on one context, every operator that shares the space in turn."""
    from volta_mi355x import Backend
    g = gen(dim)
    with Backend(timing_policy=1) as b:
        for batch in (2, 70):
            check_window(b, batch, [1] * batch, [2000 + i for i in range(batch)], 4, 2, dim, 1500, 3)
            check_prefix(b, batch, [1] * batch, [30] * batch, 8192, 4, 4, dim)
            check_choose(b, g.integers(-9999, 9999, (batch, 9000)), choice_rows(g, batch, 9000))


@pytest.mark.gpu
def test_one_call_after_another_in_the_same_space(backend):
    """The second call's launches reuse the first's space while it may still run."""
    table = exponentials()
    calls = [make(seed, [1] * 40, [50 + seed] * 40, 8, 4, 128, 4100) for seed in (1, 2)]
    got = [run(backend, *c, 13, table) for c in calls for _ in range(3)]
    for i in range(3):
        for j in (0, 1):
            assert all(np.array_equal(x, y) for x, y in zip(got[3 * j], got[3 * j + i]))


@pytest.mark.gpu
@pytest.mark.parametrize("count,heads,refused", [(1 << 24, 257, True), (1 << 24, 128, True), (32769, 65535, True),
                                                 (32767, 65535, False), (1 << 24, 127, False)])
def test_rows_that_32_bits_do_not_hold_are_refused(backend, count, heads, refused):
    """Tokens x heads of a sequence from 2^31 - 127 on, 8 GB of queries of one place: before anything else of the call is
    looked at.  (One row less is refused here for its buffers, which hold none of it.)"""
    from volta_mi355x import accel
    b = backend
    cache = b.fixed_kv_cache(2, 1, 1, 64)
    x, exp = b.upload_device(np.zeros(64, np.int16)), b.upload_device(exponentials())
    try:
        a = accel._FixedAttention(x.id, 0, heads, exp.id, 0, 8192, x.id, 0, heads, heads, 12, 0)
        s = np.array([[0, 0, count, 5]], np.int64)
        for call in (lambda: b.lib.volta_mi355x_fixed_attention_device(b.raw, cache._args(), a, s.ctypes.data, 1),
                     lambda: b.lib.volta_mi355x_fixed_prefix_attention_device(b.raw, cache._args(), a, 1, 5, s.ctypes.data, 1)):
            assert call() != 0
            assert ("32 bits" in b.last_error()) == refused, b.last_error()
    finally:
        b.free_fixed_kv_cache(cache)
        b.free_device(x)
        b.free_device(exp)
