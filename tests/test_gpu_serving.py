"""Operators that serve the committed model, on the GPU against their definitions in whole numbers
(serving_reference.py): every value has one defined rounding, so the tolerance is zero."""
import numpy as np
import pytest
import serving_reference as want
from test_gpu_fixed import Held, exponentials, full, gen, normal

pytestmark = pytest.mark.gpu


# ---- attention over a window, and behind a prefix -------------------------------------------------

def make(seed, counts, lengths, heads, kv_heads, dim, prefix=0, ends=False):
    g = gen(seed)
    one = (lambda shape, std: full(g, shape)) if ends else (lambda shape, std: normal(g, shape, std))
    q = [one((n, heads, dim), 1000) for n in counts]
    k, v = ([one((t, kv_heads, dim), std) for t in lengths] for std in (1000, 3000))
    pk, pv = (one((prefix, kv_heads, dim), std) for std in (1000, 3000))
    return q, k, v, pk, pv


def run(b, q, k, v, pk, pv, shift, table, *, capacity=None, order=None, row_gap=0, gap=0, offset=0, **kw):
    """The sequences' rows in turn, `row_gap` rows apart; slots in `order`; what the cache held before is not zero."""
    heads, dim = q[0].shape[1:]
    kv_heads = k[0].shape[1]
    n = len(q)
    capacity = capacity or max([len(t) for t in k] + [len(pk), 1])
    order = list(range(n)) if order is None else order
    slots = max(order) + 2  # the last holds the prefix
    with Held(b) as held:
        cache = b.fixed_kv_cache(slots, kv_heads, dim, capacity)
        held.keep(cache.storage)
        stale = held.new(capacity * kv_heads * dim, np.int16, 32767)
        b.fixed_kv_append_device(cache, stale, stale, [[s, 0, capacity, capacity] for s in range(slots)])
        for slot, keys, values in [(s, k[i], v[i]) for i, s in enumerate(order)] + [(slots - 1, pk, pv)]:
            if len(keys):
                b.fixed_kv_append_device(cache, held.put(keys), held.put(values), [[slot, 0, len(keys), len(keys)]])
        stride, seqs, row = heads * dim + gap, [], 0
        for i, s in enumerate(order):
            seqs.append([s, row, len(q[i]), len(k[i])])
            row += len(q[i]) + row_gap
        rows = max(row, 1)
        wide = np.full((rows, stride), 4321, np.int16)
        for (_, first, count, _), part in zip(seqs, q):
            wide[first:first + count, :heads * dim] = part.reshape(count, heads * dim)
        dq = held.put(np.concatenate([np.full(offset, 7, np.int16), wide.reshape(-1)]))
        out = held.new(offset + rows * stride, np.int16, -77)
        if len(pk):
            kw["prefix"] = (slots - 1, len(pk))
        b.fixed_attention_device(dq, cache, seqs, heads, held.put(table), shift, q_offset=offset, q_stride=stride, out=out,
                                 out_offset=offset, out_stride=stride, **kw)
        got = b.download_device(out)
        assert (got[:offset] == -77).all()
        got = got[offset:].reshape(rows, stride)
        parts = []
        for _, first, count, _ in seqs:
            parts.append(got[first:first + count, :heads * dim].reshape(count, heads, dim).copy())
            got[first:first + count, :heads * dim] = -77
        assert (got == -77).all()  # nothing beside the rows is written
        return parts


def check_window(b, seed, counts, lengths, heads, kv_heads, dim, window, sinks, *, shift=None, ends=False, entries=8192, **kw):
    q, k, v, pk, pv = make(seed, counts, lengths, heads, kv_heads, dim, ends=ends)
    table = exponentials(entries)
    shift = shift or max(8, round(np.log2(np.sqrt(dim) * 1e6 / 1280.0)))
    got = run(b, q, k, v, pk, pv, shift, table, window=window, sinks=sinks, **kw)
    for i, (m, t) in enumerate(zip(counts, lengths)):
        expect = want.attention(q[i], k[i], v[i], want.window_seen(m, t, window, sinks), table, shift)
        assert np.array_equal(got[i], expect), (i, m, t)


@pytest.mark.parametrize("dim", [1, 33, 64, 65, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 70), (63, 1), (64, 64), (65, 63), (100, 5), (300, 0), (1 << 40, 3)])
def test_window_head_sizes(backend, dim, window, sinks):
    """Prompts, single tokens and some tokens over a cache in one call."""
    check_window(backend, dim + window % 999, [130, 1, 7, 1], [130, 257, 300, 1], 3, 3, dim, window, sinks)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 1), (8, 2), (6, 3), (17, 1)])
@pytest.mark.parametrize("window,sinks", [(40, 0), (130, 4)])
def test_window_grouped_heads(backend, heads, kv_heads, window, sinks):
    check_window(backend, heads, [90, 1, 3, 33], [90, 500, 201, 133], heads, kv_heads, 48, window, sinks, order=[2, 0, 3, 1])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("length", [60, 300, 700, 1100, 2500, 5000])
@pytest.mark.parametrize("window,sinks", [(200, 4), (1024, 100), (4000, 0)])
def test_window_tokens_over_long_caches(backend, dim, length, window, sinks):
    """Windows whose tiles are few, fit LDS, and are split over workgroups."""
    check_window(backend, length + dim, [1, 2], [length, length - 3], 4, 2, dim, window, sinks)


@pytest.mark.parametrize("dim,batch,heads", [(64, 2, 12), (64, 40, 12), (128, 3, 8)])
@pytest.mark.parametrize("window,sinks", [(128, 0), (129, 66), (500, 3)])
def test_window_many_prompts(backend, dim, batch, heads, window, sinks):
    """Whole prompts, of one team of waves and of two, and heads over 64."""
    g = gen(dim + batch)
    lengths = [int(n) for n in g.integers(200, 800 if batch < 10 else 400, batch)]
    check_window(backend, batch, lengths, lengths, heads, heads // 4, dim, window, sinks)


@pytest.mark.parametrize("counts,lengths", [([1], [900]), ([20], [900]), ([200, 1], [400, 3000])])
@pytest.mark.parametrize("shift", [8, 13, 17, 24])
def test_window_values_at_the_ends(backend, counts, lengths, shift):
    check_window(backend, shift, counts, lengths, 4, 2, 64, 150, 10, shift=shift, ends=True)
    check_window(backend, shift, counts, lengths, 4, 2, 128, 150, 10, shift=shift, ends=True)


def test_window_strides_rows_apart_and_short_tables(backend):
    check_window(backend, 5, [70, 2, 1], [99, 200, 300], 4, 2, 40, 64, 65, row_gap=3, gap=5, offset=3)
    for entries in (1, 2, 77):
        check_window(backend, entries, [70, 2, 1], [99, 200, 300], 4, 2, 64, 64, 0, entries=entries)


def test_window_of_many_sequences(backend):
    g = gen(2)
    lengths = [int(n) for n in g.integers(1, 300, 150)]
    counts = [int(g.integers(0, n + 1)) for n in lengths]
    check_window(backend, 6, counts, lengths, 2, 1, 16, 50, 7)


def test_a_window_that_holds_everything_is_no_window(backend):
    q, k, v, pk, pv = make(4, [5, 1], [300, 200], 4, 2, 64)
    table = exponentials()
    one = run(backend, q, k, v, pk, pv, 13, table)
    for window, sinks in ((300, 0), (250, 50), (10, 290), (1 << 40, 0)):
        two = run(backend, q, k, v, pk, pv, 13, table, window=window, sinks=sinks)
        assert all(np.array_equal(x, y) for x, y in zip(one, two))


def check_prefix(b, seed, counts, lengths, prefix, heads, kv_heads, dim, *, causal=True, shift=None, ends=False, **kw):
    q, k, v, pk, pv = make(seed, counts, lengths, heads, kv_heads, dim, prefix, ends)
    table = exponentials()
    shift = shift or max(8, round(np.log2(np.sqrt(dim) * 1e6 / 1280.0)))
    got = run(b, q, k, v, pk, pv, shift, table, causal=causal, **kw)
    for i, (m, t) in enumerate(zip(counts, lengths)):
        expect = want.attention(q[i], np.concatenate([pk, k[i]]), np.concatenate([pv, v[i]]),
                                want.prefix_seen(m, prefix, t, causal), table, shift)
        assert np.array_equal(got[i], expect), (i, m, t)


@pytest.mark.parametrize("dim", [1, 33, 64, 65, 128])
@pytest.mark.parametrize("prefix", [1, 63, 64, 65, 200, 1000])
def test_prefix_head_sizes(backend, dim, prefix):
    check_prefix(backend, dim + prefix, [130, 1, 7, 1], [130, 257, 300, 1], prefix, 3, 3, dim)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 1), (8, 2), (6, 3), (17, 1)])
@pytest.mark.parametrize("prefix", [50, 640])
def test_prefix_grouped_heads(backend, heads, kv_heads, prefix):
    check_prefix(backend, heads, [90, 1, 3, 33], [90, 500, 201, 133], prefix, heads, kv_heads, 48, order=[2, 0, 3, 1])


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 12, 12), (64, 8, 2), (128, 8, 2), (128, 4, 4)])
@pytest.mark.parametrize("batch,new", [(1, 1), (4, 1), (33, 1), (64, 1), (70, 1), (9, 3)])
@pytest.mark.parametrize("prefix,longest", [(100, 40), (1000, 9), (3001, 300)])
def test_prefix_of_tokens_of_many_sequences(backend, dim, heads, kv_heads, batch, new, prefix, longest):
    g = gen(dim + batch)
    lengths = [int(n) for n in g.integers(new, longest + 1, batch)]
    check_prefix(backend, batch + prefix, [new] * batch, lengths, prefix, heads, kv_heads, dim)


# Few rows of many sequences behind a prefix of 33 tiles, 124 units of 16 rows: near the bounds of the rule that has them
# read it together or not.  test_serving_paths.py holds cases to each of its outcomes.
TOGETHER = dict(counts=[1] * 31, prefix=2100, kv_heads=4)


@pytest.mark.parametrize("dim", [1, 33, 64, 65, 128])
@pytest.mark.parametrize("heads", [4, 12, 64])
@pytest.mark.parametrize("prefix", [2049, 2111, 2112])
def test_prefix_read_together(backend, dim, heads, prefix):
    g = gen(dim + heads)
    check_prefix(backend, prefix, TOGETHER["counts"], [int(n) for n in g.integers(1, 200, 31)], prefix, heads, 4, dim)


@pytest.mark.parametrize("dim", [40, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_prefix_read_together_by_different_counts_rows_apart(backend, dim, causal):
    g = gen(dim)
    counts = [int(n) for n in g.integers(0, 4, 50)]
    lengths = [max(n, int(m)) if causal else int(m) for n, m in zip(counts, g.integers(0, 300, 50))]
    order = [int(i) for i in g.permutation(50)]
    check_prefix(backend, dim, counts, lengths, 2100, 12, 4, dim, causal=causal, row_gap=2, gap=3, offset=1, order=order)
    check_prefix(backend, dim + 1, [2] * 40, [n + 2 for n in lengths[:40]], 2100, 8, 4, dim, causal=causal, row_gap=1)


@pytest.mark.parametrize("shift", [8, 13, 17, 24])
@pytest.mark.parametrize("dim", [64, 128])
def test_prefix_read_together_with_values_at_the_ends(backend, shift, dim):
    g = gen(shift)
    check_prefix(backend, shift, TOGETHER["counts"], [int(n) for n in g.integers(1, 100, 31)], 2100, 8, 4, dim, shift=shift,
                 ends=True)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch", [63, 64, 65, 130, 192])
def test_prefix_read_together_by_launches_of_64_sequences(backend, dim, batch):
    g = gen(batch)
    check_prefix(backend, batch, [1] * batch, [int(n) for n in g.integers(1, 90, batch)], 2000, 4, 4, dim)


def test_prefix_read_together_beside_prompts(backend):
    """Sequences of few rows and of many in one call."""
    g = gen(4)
    counts = [1, 200, 1, 90] + [1] * 40
    lengths = [50, 200, 1, 130] + [int(n) for n in g.integers(1, 70, 40)]
    check_prefix(backend, 8, counts, lengths, 2200, 8, 4, 64)
    check_prefix(backend, 8, counts, lengths, 2200, 4, 4, 96)


def test_prefix_read_together_longest_sums_of_equal_values(backend):
    """65,536 keys of the same score with exponentials of 2^14 and values at the end: sums of a part near 2^31."""
    for value in (32767, -32768):
        q = [np.full((1, 2, 3), 100, np.int16) for _ in range(2)]
        k = [np.full((n, 2, 3), 100, np.int16) for n in (1000, 36)]
        v = [np.full((n, 2, 3), value, np.int16) for n in (1000, 36)]
        pk, pv = np.full((64500, 2, 3), 100, np.int16), np.full((64500, 2, 3), value, np.int16)
        got = run(backend, q, k, v, pk, pv, 13, np.full(4, 1 << 14, np.uint16))
        assert all((part == value).all() for part in got)


@pytest.mark.parametrize("dim,batch", [(64, 3), (64, 20), (128, 4)])
@pytest.mark.parametrize("prefix", [64, 777])
def test_prefix_of_many_prompts(backend, dim, batch, prefix):
    g = gen(dim + batch)
    lengths = [int(n) for n in g.integers(40, 500, batch)]
    check_prefix(backend, batch, lengths, lengths, prefix, 6, 3, dim)


@pytest.mark.parametrize("causal", [True, False])
def test_prefix_with_sequences_of_no_tokens(backend, causal):
    """Rows that see the prefix alone (not causal), and sequences without rows."""
    counts, lengths = ([0, 5, 0, 1], [3, 9, 0, 1]) if causal else ([2, 5, 0, 20], [0, 3, 0, 1])
    check_prefix(backend, 3, counts, lengths, 130, 4, 2, 64, causal=causal)
    check_prefix(backend, 3, counts, lengths, 130, 4, 2, 128, causal=causal)


@pytest.mark.parametrize("counts,lengths", [([1] * 3, [1, 70, 30]), ([20], [90]), ([200, 1], [400, 30])])
@pytest.mark.parametrize("shift", [8, 13, 17, 24])
def test_prefix_values_at_the_ends(backend, counts, lengths, shift):
    check_prefix(backend, shift, counts, lengths, 333, 4, 2, 64, shift=shift, ends=True)
    check_prefix(backend, shift, counts, lengths, 333, 4, 2, 128, shift=shift, ends=True)


def test_prefix_strides_and_rows_apart(backend):
    check_prefix(backend, 5, [70, 2, 1], [99, 200, 30], 99, 4, 2, 40, row_gap=3, gap=5, offset=3)
    check_prefix(backend, 6, [1] * 40, [9] * 40, 500, 4, 2, 64, row_gap=1, gap=1, offset=1)


def test_a_prefix_equals_the_same_tokens_in_each_sequence(backend):
    q, k, v, pk, pv = make(9, [1, 4, 50], [20, 4, 90], 4, 2, 64, 300)
    table = exponentials()
    one = run(backend, q, k, v, pk, pv, 13, table)
    none = pk[:0]
    two = run(backend, q, [np.concatenate([pk, t]) for t in k], [np.concatenate([pv, t]) for t in v], none, none, 13, table)
    assert all(np.array_equal(x, y) for x, y in zip(one, two))


# ---- heads normed and rotated -----------------------------------------------------------------------

def run_rotate(b, x, heads, kv_heads, dim, *, x_gap=0, out_gap=0, offset=0, in_place=False, **kw):
    rows, cols = x.shape
    with Held(b) as held:
        wide = np.full((rows, cols + x_gap), 1234, np.int16)
        wide[:, :cols] = x
        dx = held.put(np.concatenate([np.full(offset, -5, np.int16), wide.reshape(-1)]))
        args = dict(kw)
        for name in ("q_gain", "k_gain", "angles", "positions"):
            args[name] = held.put(kw.get(name))
        if kw.get("angles") is not None:
            args["angle_rows"] = len(kw["angles"])
        if in_place:
            b.fixed_rotate_device(dx, rows, heads, dim, kv_heads=kv_heads, x_offset=offset, x_stride=cols + x_gap, out=dx,
                                  out_offset=offset, out_stride=cols + x_gap, **args)
            got = b.download_device(dx)
            assert (got[:offset] == -5).all()
            got = got[offset:].reshape(rows, -1)
            assert (got[:, cols:] == 1234).all()
            return got[:, :cols]
        out = held.new(offset + rows * (cols + out_gap), np.int16, 99)
        b.fixed_rotate_device(dx, rows, heads, dim, kv_heads=kv_heads, x_offset=offset, x_stride=cols + x_gap, out=out,
                              out_offset=offset, out_stride=cols + out_gap, **args)
        got = b.download_device(out)
        assert (got[:offset] == 99).all()
        got = got[offset:].reshape(rows, -1)
        assert (got[:, cols:] == 99).all()
        return got[:, :cols]


def check_rotate(b, seed, rows, heads, kv_heads, dim, rotated, *, gains=True, ends=False, places=50, adjacent=False,
                 gain_shift=2, eps=1, angle_shift=14, **kw):
    g = gen(seed)
    one = (lambda shape, std: full(g, shape)) if ends else (lambda shape, std: normal(g, shape, std))
    x = one((rows, (heads + kv_heads) * dim), 1500)
    x[g.random(rows) < 0.1] = 0  # a head of zeros stays zeros
    args = dict(gain_shift=gain_shift, eps=eps, angle_shift=angle_shift, adjacent=adjacent, rotated=rotated)
    if gains:
        args.update(q_gain=one(dim, 4000), k_gain=one(dim, 4000))
    if rotated:
        # positions before and behind the table too
        args.update(angles=one((places, rotated // 2, 2), 9000), positions=g.integers(-2, places + 2, rows).astype(np.int32))
    expect = want.rotate(x, heads, dim, **args)
    assert np.array_equal(run_rotate(b, x, heads, kv_heads, dim, **args, **kw), expect)


@pytest.mark.parametrize("dim", [1, 2, 3, 8, 17, 31, 32, 33, 40, 64, 65, 80, 96, 127, 128])
@pytest.mark.parametrize("adjacent", [False, True])
def test_rotate_head_sizes(backend, dim, adjacent):
    for rotated in sorted({0, 2 * (dim // 4), 2 * (dim // 2), min(2 * (dim // 2), 6)}):
        for gains in (False, True):
            check_rotate(backend, dim + rotated, 9, 3, 2, dim, rotated, gains=gains, adjacent=adjacent)


@pytest.mark.parametrize("rows,heads,kv_heads", [(1, 12, 12), (1, 1, 0), (3, 0, 5), (257, 5, 1), (1000, 12, 4)])
def test_rotate_rows_and_heads(backend, rows, heads, kv_heads):
    check_rotate(backend, rows, rows, heads, kv_heads, 64, 64)
    check_rotate(backend, rows + 1, rows, heads, kv_heads, 128, 96, adjacent=True)


@pytest.mark.parametrize("dim,rotated", [(5, 4), (64, 64), (128, 128), (80, 40)])
@pytest.mark.parametrize("adjacent", [False, True])
def test_rotate_values_at_the_ends(backend, dim, rotated, adjacent):
    for gain_shift, eps, angle_shift in ((0, 1, 0), (15, 1 << 40, 15), (3, 7, 14)):
        check_rotate(backend, dim, 33, 3, 2, dim, rotated, ends=True, adjacent=adjacent, gain_shift=gain_shift, eps=eps,
                     angle_shift=angle_shift)


@pytest.mark.parametrize("a,b_,c,s", [(-32768, -32768, -32768, 32767), (-32768, 32767, 32767, -32768),
                                      (-32768, -32768, -32768, -32768), (32767, 32767, 32767, 32767)])
def test_rotate_sums_of_the_largest_products(backend, a, b_, c, s):
    """a c - b s and a s + b c reach 2^31 and -2^31 + 2^16."""
    x = np.tile(np.array([a, b_], np.int16), (4, 32))
    angles = np.tile(np.array([c, s], np.int16), (2, 32, 1))
    for shift in (0, 14, 15):
        kw = dict(angles=angles, positions=np.array([0, 1, 0, 1], np.int32), rotated=64, adjacent=True, angle_shift=shift)
        assert np.array_equal(run_rotate(backend, x, 1, 0, 64, **kw), want.rotate(x, 1, 64, **kw))


@pytest.mark.parametrize("x_gap,out_gap,offset", [(0, 0, 1), (1, 2, 3), (64, 0, 0), (7, 13, 5)])
@pytest.mark.parametrize("dim,rotated", [(64, 64), (40, 22), (33, 10)])
def test_rotate_strides_alignment_and_in_place(backend, x_gap, out_gap, offset, dim, rotated):
    for adjacent in (False, True):
        for in_place in (False, True):
            check_rotate(backend, dim, 37, 3, 1, dim, rotated, adjacent=adjacent, x_gap=x_gap, out_gap=out_gap, offset=offset,
                         in_place=in_place)


def test_rotate_one_gain_alone(backend):
    g = gen(8)
    x, gain = normal(g, (20, 4 * 64), 1500), normal(g, 64, 4000)
    for kw in (dict(q_gain=gain), dict(k_gain=gain)):
        kw = dict(kw, gain_shift=3, eps=5, rotated=0)
        assert np.array_equal(run_rotate(backend, x, 3, 1, 64, **kw), want.rotate(x, 3, 64, **kw))


def test_rotate_equals_the_norm_of_each_head(backend):
    g = gen(11)
    x, gain = normal(g, (50, 64), 1500), normal(g, 64, 4000)
    with Held(backend) as held:
        dx, dg, out = held.put(x), held.put(gain), held.new(50 * 64, np.int16)
        backend.fixed_norm_device(dx, 50, 64, dg, 2, 4096, rms=True, out=out)
        norm = backend.download_device(out)
        backend.fixed_rotate_device(dx, 50, 1, 64, q_gain=dg, gain_shift=2, eps=4096, out=out)
        assert np.array_equal(backend.download_device(out), norm)


# ---- the choice of a token ----------------------------------------------------------------------------

def run_choose(b, logits, rows, *, bias_shift=0, gap=0, offset=0, adjusted="new", mask_gap=0, junk=0):
    """rows as in the reference; lists packed with `junk` entries before each."""
    from volta_mi355x import FIXED_CHOICE
    n, vocab = logits.shape
    words = (vocab + 31) // 32
    choices = np.zeros(n, FIXED_CHOICE)
    history, tokens, values, masks = [], [], [], []
    for i, r in enumerate(rows):
        history += [0] * junk
        tokens += [0] * junk
        values += [99] * junk
        choices[i] = (len(history), len(r["history"]), len(tokens), len(r["biases"]), -1 if r["mask"] is None else len(masks),
                      r["frequency"], r["presence"], r["repetition"], 0)
        history += list(r["history"])
        tokens += [t for t, _ in r["biases"]]
        values += [v for _, v in r["biases"]]
        if r["mask"] is not None:
            bits = np.packbits(np.pad(r["mask"], (0, words * 32 - vocab), constant_values=True), bitorder="little")
            masks.append(np.concatenate([bits.view("<u4"), np.full(mask_gap, 0x5555AAAA, "<u4")]))
    with Held(b) as held:
        wide = np.full((n, vocab + gap), (1 << 62), np.int64)
        wide[:, :vocab] = logits
        dl = held.put(np.concatenate([np.full(offset, 1 << 62, np.int64), wide.reshape(-1)]))
        put = lambda a, dtype: held.put(np.array(a, dtype)) if len(a) else None
        kw = dict(history=put(history, np.int32), bias_tokens=put(tokens, np.int32), bias_values=put(values, np.int32),
                  allowed=held.put(np.concatenate(masks)) if masks else None, allowed_stride=words + mask_gap)
        da = None
        if adjusted == "in place":
            da = dl
        elif adjusted == "new":
            da = held.new(offset + n * (vocab + gap), np.int64, 55)
        if da is not None:
            kw.update(adjusted=da, adjusted_offset=offset, adjusted_stride=vocab + gap)
        out = held.new(n + 2, np.int32, 77)
        b.fixed_choose_device(dl, n, vocab, choices, bias_shift=bias_shift, logits_offset=offset, logits_stride=vocab + gap,
                              out=out, out_offset=1, **kw)
        got = b.download_device(out)
        assert got[0] == 77 and got[-1] == 77
        if da is None:
            return got[1:-1], None
        full_out = b.download_device(da)
        beside = 1 << 62 if adjusted == "in place" else 55
        assert (full_out[:offset] == beside).all()
        full_out = full_out[offset:].reshape(n, -1)
        assert (full_out[:, vocab:] == beside).all()
        return got[1:-1], full_out[:, :vocab]


def choice_rows(g, rows, vocab, history=20, biases=5, masked=0.5):
    out = []
    for _ in range(rows):
        pool = g.integers(-3, vocab + 3, max(1, history // 2))  # tokens outside the vocabulary too, many twice
        out.append(dict(history=g.choice(pool, int(g.integers(0, history + 1))),
                        biases=[(int(t), int(v)) for t, v in zip(g.choice(pool, biases), g.integers(-999, 999, biases))],
                        mask=g.random(vocab) < 0.7 if g.random() < masked else None,
                        frequency=int(g.integers(-50, 200)), presence=int(g.integers(-50, 300)),
                        repetition=int(g.choice([65536, 78643, 60000, 1, (1 << 32) - 1]))))
    return out


def check_choose(b, logits, rows, **kw):
    shift = kw.get("bias_shift", 0)
    tokens, adjusted = want.choose(logits, rows, bias_shift=shift)
    got, out = run_choose(b, logits, rows, **kw)
    assert np.array_equal(got, tokens)
    if out is not None:
        assert np.array_equal(out, adjusted)


@pytest.mark.parametrize("vocab", [1, 2, 31, 32, 33, 511, 2047, 2048, 2049, 4095, 4097, 8193, 16385, 50257])
@pytest.mark.parametrize("rows", [1, 3])
def test_choose_vocabularies(backend, vocab, rows):
    g = gen(vocab)
    logits = np.rint(g.normal(0, 3000, (rows, vocab))).astype(np.int64)
    for adjusted in ("new", "in place", None):
        check_choose(backend, logits, choice_rows(g, rows, vocab), adjusted=adjusted, bias_shift=3)


@pytest.mark.parametrize("rows", [63, 64, 65, 200, 300])
def test_choose_many_rows(backend, rows):
    g = gen(rows)
    logits = np.rint(g.normal(0, 3000, (rows, 2500))).astype(np.int64)
    check_choose(backend, logits, choice_rows(g, rows, 2500, history=60, biases=11), junk=3, mask_gap=2)


def test_choose_more_rows_than_a_launch_takes(backend):
    g = gen(8200)
    logits = np.rint(g.normal(0, 3000, (8200, 5))).astype(np.int64)
    check_choose(backend, logits, choice_rows(g, 8200, 5, history=4, biases=2), mask_gap=1, gap=2, adjusted="new")


@pytest.mark.parametrize("bias_shift", [0, 30, 46])
def test_choose_logits_at_the_ends(backend, bias_shift):
    """Products and sums far beyond 64 bits, clamped once."""
    g = gen(5 + bias_shift)
    logits = g.choice(np.array([-(1 << 63), -(1 << 63) + 1, (1 << 63) - 1, (1 << 62), -1, 0, 1, 12345], np.int64), (8, 700))
    rows = choice_rows(g, 8, 700, history=900, biases=200)
    for r, f in zip(rows, ((1 << 63) - 1, -(1 << 63), 1 << 40, -5, 0, 1 << 62, 3, -(1 << 50))):
        r["frequency"], r["presence"] = f, -f - 1
        r["biases"] = [(t, int(g.choice([-(1 << 31), (1 << 31) - 1, 1, 0]))) for t, _ in r["biases"]]
    check_choose(backend, logits, rows, bias_shift=bias_shift)


@pytest.mark.parametrize("repetition", [1, 2, 3, 65535, 65536, 65537, 98304, (1 << 31) + 1, (1 << 32) - 1])
def test_choose_repetition_rounding(backend, repetition):
    g = gen(repetition)
    logits = np.concatenate([np.arange(-600, 600), g.integers(-(1 << 62), 1 << 62, 800)]).astype(np.int64)[None]
    rows = [dict(history=np.arange(2000), biases=[], mask=None, frequency=0, presence=0, repetition=repetition)]
    check_choose(backend, logits, rows)


@pytest.mark.parametrize("vocab", [100, 2048, 9000])
def test_choose_ties_go_to_the_lowest_index(backend, vocab):
    g = gen(vocab)
    plain = dict(history=[], biases=[], mask=None, frequency=0, presence=0, repetition=65536)
    logits = np.full((4, vocab), -7, np.int64)
    logits[1, vocab // 2:] = 3
    logits[2, [vocab - 1, vocab - 2]] = 9
    logits[3] = -(1 << 63)
    check_choose(backend, logits, [plain] * 4)
    check_choose(backend, logits, [dict(plain, mask=g.random(vocab) < 0.1) for _ in range(4)])


@pytest.mark.parametrize("vocab", [1, 70, 5000])
def test_choose_masks_that_leave_one_token_or_none(backend, vocab):
    g = gen(vocab)
    logits = g.integers(-9, 9, (5, vocab))
    logits[2] = (1 << 63) - 1
    masks = [np.zeros(vocab, bool) for _ in range(5)]
    masks[1][vocab - 1] = masks[3][0] = masks[4][vocab // 2] = True
    rows = [dict(history=[vocab - 1] * 3, biases=[(0, -(1 << 31))], mask=m, frequency=(1 << 63) - 1, presence=9,
                 repetition=70000) for m in masks]
    check_choose(backend, logits, rows, bias_shift=46)


def test_choose_long_histories(backend):
    g = gen(3)
    logits = np.rint(g.normal(0, 1e6, (3, 6000))).astype(np.int64)
    rows = choice_rows(g, 3, 6000)
    for r, n in zip(rows, (70000, 8191, 300)):
        r["history"] = (g.random(n) ** 3 * 6000).astype(np.int64)
        r["biases"] = [(int(t), 3) for t in g.integers(0, 6000, 3000)]
        r["frequency"] = 17
    check_choose(backend, logits, rows, bias_shift=2, gap=5, offset=3)


@pytest.mark.parametrize("repetition", [(1 << 15) - 1, 1 << 15, (1 << 15) + 1, 70001, (1 << 17) - 1, 1 << 17, (1 << 17) + 1])
def test_choose_where_doubles_and_64_bits_end(backend, repetition):
    """Logits, frequencies, presences and biases at the ends of what the shorter arithmetic holds, in rows of their own."""
    g = gen(repetition)
    end, rows, logits = 1 << 35, [], []
    for top in (end - 1, end, end + 1):
        for frequency, presence in ((0, 0), ((1 << 31) - 1, (1 << 55) - 1), (-(1 << 31) + 1, -(1 << 55) + 1), (1 << 31, 5),
                                    (-(1 << 31), 1 << 55)):
            logits.append(g.choice([top, -top, top - 1, 1 - top, 12345, -54321, 0, -1], 300))
            rows.append(dict(history=g.integers(0, 300, 500), mask=None, frequency=frequency, presence=presence,
                             repetition=repetition, biases=[(int(i), int(v)) for i, v in zip(
                                 g.integers(0, 300, 40), g.choice([1, -1, (1 << 31) - 1, -(1 << 31)], 40))]))
    logits = np.array(logits, np.int64)
    for shift in (0, 10, 29, 30, 46):
        check_choose(backend, logits, rows, bias_shift=shift)


@pytest.mark.parametrize("biases", [511, 512, 513, 1500])
def test_choose_many_biases(backend, biases):
    """Biases of as many tokens as the table holds, of more, and several of a token."""
    g = gen(biases)
    rows = choice_rows(g, 2, 5000)
    for r in rows:
        r["biases"] = [(int(i), int(v)) for i, v in zip(g.permutation(5000)[:biases], g.integers(-9999, 9999, biases))]
    rows[1]["biases"] = [(i % 400, v) for i, v in rows[1]["biases"]]
    check_choose(backend, np.rint(g.normal(0, 3000, (2, 5000))).astype(np.int64), rows, bias_shift=1)


@pytest.mark.parametrize("history", [32767, 32768])
def test_choose_one_token_that_often(backend, history):
    g = gen(history)
    rows = [dict(history=[77] * history, biases=[(77, 5), (78, 6)], mask=None, frequency=3, presence=1, repetition=66000)]
    check_choose(backend, g.integers(-10 ** 6, 10 ** 6, (1, 200)), rows)


@pytest.mark.parametrize("vocab", [1, 2815, 2816, 2817, 20480, 20481, 60001])
@pytest.mark.parametrize("biases", [0, 512, 513, 2048, 2049, 5000])
@pytest.mark.parametrize("rows", [2, 70])
def test_choose_lists_beyond_the_short_ones(backend, vocab, biases, rows):
    """Histories that 15 bits do not count, more biases than half a table holds, on the edges of their chunks."""
    g = gen(vocab + biases)
    some = choice_rows(g, rows, vocab, history=30, biases=20)
    for r in (some[0], some[-1]):
        r["history"] = np.concatenate([np.full(32768, vocab // 2), g.integers(0, vocab, 900)])
        r["biases"] = [(int(t), int(v)) for t, v in zip(g.integers(-3, vocab + 3, biases), g.integers(-9999, 9999, biases))]
    check_choose(backend, np.rint(g.normal(0, 9000, (rows, vocab))).astype(np.int64), some, bias_shift=4)


@pytest.mark.parametrize("vocab", [57343, 57344, 57345, 130001])
def test_choose_rows_of_the_largest_chunks(backend, vocab):
    """A workgroup a chunk of up to 57,344 tokens, of as many rows as there are CUs; three rows have lists."""
    g = gen(vocab)
    n = 256
    logits = g.integers(-(1 << 30), 1 << 30, (n, vocab))
    plain = dict(history=[], biases=[], mask=None, frequency=0, presence=0, repetition=65536)
    rows = [plain] * n
    some = [0, 100, 255]
    for i, r in zip(some, choice_rows(g, 3, vocab, history=9000, biases=100)):
        rows[i] = r
    tokens, adjusted = logits.argmax(1), logits.copy()
    tokens[some], adjusted[some] = want.choose(logits[some], [rows[i] for i in some], bias_shift=9)
    got, out = run_choose(backend, logits, rows, bias_shift=9)
    assert np.array_equal(got, tokens) and np.array_equal(out, adjusted)


@pytest.mark.parametrize("vocab", [20479, 20480, 20481, 61440])
@pytest.mark.parametrize("history,biases", [(33000, 100), (9000, 2048), (40000, 2100)])
def test_choose_rows_of_the_largest_chunks_of_long_lists(backend, vocab, history, biases):
    """The same with counts of 31 bits: chunks of up to 20,480 tokens, or of 2,816 where biases are many."""
    g = gen(vocab + history)
    n = 256
    logits = g.integers(-(1 << 30), 1 << 30, (n, vocab))
    plain = dict(history=[], biases=[], mask=None, frequency=0, presence=0, repetition=65536)
    rows = [plain] * n
    some = [1, 255]
    for i, r in zip(some, choice_rows(g, 2, vocab)):
        rows[i] = r
        r["history"] = np.concatenate([np.full(history - 500, vocab - 1), g.integers(0, vocab, 500)])
        r["biases"] = [(int(t), int(v)) for t, v in zip(g.permutation(vocab)[:biases], g.integers(-9999, 9999, biases))]
    tokens, adjusted = logits.argmax(1), logits.copy()
    tokens[some], adjusted[some] = want.choose(logits[some], [rows[i] for i in some], bias_shift=9)
    got, out = run_choose(backend, logits, rows, bias_shift=9)
    assert np.array_equal(got, tokens) and np.array_equal(out, adjusted)


def test_choose_without_choices_is_the_largest(backend):
    g = gen(1)
    logits = g.integers(-99, 99, (70, 4000))
    with Held(backend) as held:
        out = held.keep(backend.fixed_choose_device(held.put(logits), 70, 4000))
        assert np.array_equal(backend.download_device(out), np.argmax(logits, 1))


def test_choose_without_workspaces_in_a_coarse_scope():
    from volta_mi355x import Backend
    g = gen(12)
    logits = g.integers(-9999, 9999, (3, 20000))
    with Backend(timing_policy=1) as b, Held(b) as held:
        dl, out = held.put(logits), held.new(3, np.int32)
        live = b.get_stats()["live_device_bytes"]
        assert b.lib.volta_cuda_begin_coarse_timing(b.raw, 0) == 0
        b.fixed_choose_device(dl, 3, 20000, out=out)
        assert b.lib.volta_cuda_end_coarse_timing(b.raw) == 0
        assert b.get_stats()["live_device_bytes"] == live
        assert np.array_equal(b.download_device(out), np.argmax(logits, 1))


# ---- refusals ---------------------------------------------------------------------------------------------

def test_refusals_of_the_library(backend):
    """What only the library can see: slots, lengths and overlaps."""
    from volta_mi355x import FIXED_CHOICE, GpuError
    b = backend
    with Held(b) as held:
        x, exp, out = held.new(4096, np.int16), held.put(exponentials()), held.new(4096, np.int16)
        cache = b.fixed_kv_cache(3, 2, 16, 70)
        held.keep(cache.storage)
        long = b.fixed_kv_cache(2, 1, 1, 65536)
        held.keep(long.storage)
        l, i32 = held.new(4000, np.int64), held.new(100, np.int32)
        one = np.zeros(2, FIXED_CHOICE)
        one["mask"], one["repetition"], one["history_count"] = -1, 65536, 50
        refused = [
            lambda: b.fixed_attention_device(x, cache, [[0, 0, 1, 1]], 2, exp, 12, prefix=(0, 5), out=out),
            lambda: b.fixed_attention_device(x, cache, [[1, 0, 1, 1], [0, 1, 1, 1]], 2, exp, 12, prefix=(0, 5), out=out),
            lambda: b.fixed_attention_device(x, cache, [[1, 0, 2, 1]], 2, exp, 12, prefix=(0, 5), out=out),
            lambda: b.fixed_attention_device(x, cache, [[1, 0, 1, 71]], 2, exp, 12, prefix=(0, 5), out=out),
            lambda: b.fixed_attention_device(x, cache, [[3, 0, 1, 1]], 2, exp, 12, prefix=(0, 5), out=out),
            lambda: b.fixed_attention_device(x, cache, [[0, 0, 1, 1]], 2, exp, 12, window=5, out=x),
            lambda: b.fixed_attention_device(x, cache, [[0, 0, 2, 1]], 2, exp, 12, window=5, out=out),
            lambda: b.fixed_attention_device(x, long, [[1, 0, 1, 36]], 1, exp, 12, prefix=(0, 65501), out=out),
            lambda: b.fixed_rotate_device(x, 2, 2, 16, out=x, out_offset=1),
            lambda: b.fixed_rotate_device(x, 2, 2, 16, q_gain=out, out=out),
            lambda: b.fixed_rotate_device(x, 2, 2, 16, k_gain=out, kv_heads=1, k_gain_offset=95, out=out),
            lambda: b.fixed_rotate_device(x, 2, 2, 16, angles=out, angle_rows=2, positions=i32, out=out),
            lambda: b.fixed_choose_device(l, 2, 100, adjusted=l, adjusted_offset=8),
            lambda: b.fixed_choose_device(l, 2, 100, adjusted=l, adjusted_stride=101),
            lambda: b.fixed_choose_device(l, 2, 100, one, history=i32, out=i32, out_offset=49),
        ]
        for i, call in enumerate(refused):
            try:
                call()
            except GpuError:
                continue
            pytest.fail(f"call {i} was not refused")
        # what is just inside
        b.fixed_attention_device(x, long, [[1, 0, 0, 36]], 1, exp, 12, prefix=(0, 65500), out=out)
        b.fixed_attention_device(x, cache, [[0, 0, 1, 1]], 2, exp, 12, prefix=(0, 0), out=out)
        b.fixed_choose_device(l, 2, 100, one, history=i32, out=i32, out_offset=50)
        b.fixed_choose_device(l, 2, 100, adjusted=l, adjusted_offset=200)


def test_refusals_at_the_c_entry(backend):
    import ctypes

    from volta_mi355x import accel
    b, lib = backend, backend.lib
    with Held(b) as held:
        x, i32, l = held.new(256, np.int16), held.new(8, np.int32), held.new(64, np.int64)

        def rotate(**kw):
            a = accel._FixedRotate(x_id=x.id, x_stride=32, angles_id=x.id, angle_rows=2, positions_id=i32.id,
                                   out_id=held.new(256, np.int16).id, out_stride=32, rows=4, heads=1, kv_heads=1, dim=16,
                                   rotated=16, eps=1, angle_shift=14)
            for name, value in kw.items():
                setattr(a, name, value)
            return lib.volta_mi355x_fixed_rotate_device(b.raw, ctypes.byref(a))

        assert rotate() == 0
        for kw in (dict(x_id=0), dict(x_id=999), dict(x_stride=31), dict(rows=0), dict(rows=9), dict(rows=1 << 63), dict(dim=0),
                   dict(dim=1 << 40), dict(heads=1 << 62), dict(heads=0, kv_heads=0), dict(x_off=1 << 63), dict(rotated=15),
                   dict(rotated=18), dict(rotated=0), dict(angles_id=0), dict(positions_id=0), dict(angle_rows=0),
                   dict(angle_rows=1 << 62), dict(angle_rows=17), dict(angles_off=240), dict(positions_off=5), dict(eps=0),
                   dict(eps=1 << 41), dict(gain_shift=16), dict(angle_shift=16), dict(q_gain_id=x.id, q_gain_off=250),
                   dict(out_id=x.id, out_off=1), dict(out_id=x.id, out_stride=33), dict(out_stride=31), dict(out_id=0)):
            assert rotate(**kw) != 0, kw
            assert b.last_error(), kw
        assert rotate() == 0 and rotate(rotated=0, angles_id=0, positions_id=0) == 0

        def choose(choice=None, count=2, **kw):
            rows = np.zeros(2, accel.FIXED_CHOICE)
            rows["mask"], rows["repetition"] = -1, 65536
            for name, value in (choice or {}).items():
                rows[name] = value
            a = accel._FixedChoose(logits_id=l.id, logits_stride=32, out_id=held.new(2, np.int32).id, vocab=32,
                                   history_id=i32.id, bias_tokens_id=i32.id, bias_values_id=i32.id, allowed_id=i32.id,
                                   allowed_stride=1)
            for name, value in kw.items():
                setattr(a, name, value)
            return lib.volta_mi355x_fixed_choose_device(b.raw, ctypes.byref(a), rows.ctypes.data, count)

        listed = dict(history_count=8, bias_count=8, mask=1)
        assert choose() == 0 and choose(listed) == 0
        for choice, kw in ((None, dict(count=0)), (None, dict(count=1 << 25)), (None, dict(vocab=0)), (None, dict(vocab=1 << 25)),
                           (None, dict(logits_stride=31)), (None, dict(logits_off=1)), (None, dict(logits_id=0)),
                           (None, dict(bias_shift=47)), (None, dict(out_off=1)), (None, dict(out_id=l.id)),
                           (None, dict(adjusted_id=l.id, adjusted_off=1, adjusted_stride=31)),
                           (None, dict(allowed_stride=0)), (dict(repetition=0), {}), (dict(history_count=9), {}),
                           (dict(history_first=8, history_count=1), {}), (dict(history_first=(1 << 64) - 1, history_count=1), {}),
                           (dict(history_first=(1 << 62), history_count=1), {}), (dict(history_count=1 << 25), {}),
                           (listed, dict(history_id=0)), (listed, dict(bias_tokens_id=0)), (listed, dict(bias_values_id=0)),
                           (listed, dict(allowed_id=0)), (listed, dict(allowed_id=999)), (dict(bias_count=9), {}),
                           (dict(bias_first=1 << 63, bias_count=1), {}), (dict(mask=8), {}), (dict(mask=(1 << 63) - 1), {}),
                           (dict(mask=3), dict(allowed_stride=1 << 62)), (listed, dict(out_id=i32.id))):
            assert choose(choice, **kw) != 0, (choice, kw)
            assert b.last_error(), (choice, kw)
        assert choose(listed) == 0

        cache = b.fixed_kv_cache(2, 1, 16, 64)
        held.keep(cache.storage)
        exp = held.put(exponentials())
        a = accel._FixedAttention(x.id, 0, 16, exp.id, 0, 8192, held.new(256, np.int16).id, 0, 16, 1, 12, 1)
        s = np.array([[0, 0, 1, 1]], np.int64)
        at = (ctypes.byref(cache._args()), ctypes.byref(a))
        window, prefix = lib.volta_mi355x_fixed_window_attention_device, lib.volta_mi355x_fixed_prefix_attention_device
        assert window(b.raw, *at, 1, 0, s.ctypes.data, 1) == 0 and window(b.raw, *at, 1 << 63, 1 << 63, s.ctypes.data, 1) == 0
        assert window(b.raw, *at, 0, 4, s.ctypes.data, 1) != 0
        assert prefix(b.raw, *at, 1, 64, s.ctypes.data, 1) == 0
        for slot, length in ((0, 1), (2, 1), (1 << 32, 1), (1, 65), (1, 1 << 63)):
            assert prefix(b.raw, *at, slot, length, s.ctypes.data, 1) != 0, (slot, length)
        a.causal = 0
        assert window(b.raw, *at, 1, 0, s.ctypes.data, 1) != 0
