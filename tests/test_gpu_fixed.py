"""Fixed-point model operators on the GPU against their definitions in 64-bit
integers (fixed_reference.py), bit for bit: every value is a whole number with
one defined rounding, so the tolerance is zero."""
import fixed_reference as ref
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ENTRIES = 8192


def gen(seed):
    return np.random.Generator(np.random.PCG64(seed))


def full(g, shape):
    """All of i16, its ends included often."""
    a = g.integers(-32768, 32768, size=shape, dtype=np.int64)
    ends = g.random(shape)
    a[ends < 0.1] = -32768
    a[ends > 0.9] = 32767
    return a.astype(np.int16)


def normal(g, shape, std):
    return np.clip(np.rint(g.normal(0, std, shape)), -32768, 32767).astype(np.int16)


def exponentials(entries=ENTRIES, scale=640.0):
    return np.rint(16384.0 * np.exp(-np.arange(entries) / scale)).astype(np.uint16)


class Held:
    """Uploads that go back to the pool together."""

    def __init__(self, b):
        self.b, self.bufs = b, []

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for buf in self.bufs:
            self.b.free_device(buf)

    def keep(self, buf):
        self.bufs.append(buf)
        return buf

    def put(self, a):
        return None if a is None else self.keep(self.b.upload_device(np.ascontiguousarray(a).reshape(-1)))

    def new(self, n, dtype, fill=None):
        return self.put(np.full(n, 0 if fill is None else fill, dtype))


# ---- matrix product -------------------------------------------------------------------------

def run_linear(b, x, w, *, x_gap=0, x_offset=0, out_gap=0, residual_gap=0, transposed=False, **kw):
    """The library's product, with rows x_gap, out_gap and residual_gap longer than their matrices."""
    rows, k = x.shape
    n = w.shape[1]
    raw = kw.get("raw", False)
    with Held(b) as held:
        wide = np.full((rows, k + x_gap), 12345, np.int16)
        wide[:, :k] = x
        dx = held.put(np.concatenate([np.full(x_offset, 777, np.int16), wide.reshape(-1)]))
        dw = held.put(w.T if transposed else w)
        packed = b.fixed_weights_device(dw, k, n, transposed=transposed)
        held.keep(packed.storage)
        args = dict(kw)
        for name in ("bias", "table"):
            args[name] = held.put(kw.get(name))
        if kw.get("residual") is not None:
            wide = np.full((rows, n + residual_gap), -9, np.int16)
            wide[:, :n] = kw["residual"]
            args.update(residual=held.put(wide), residual_stride=n + residual_gap)
        stride = n + out_gap
        out = held.new(rows * stride, np.int64 if raw else np.int16, 31)
        b.fixed_linear_device(dx, rows, packed, x_offset=x_offset, x_stride=k + x_gap, out=out, out_stride=stride, **args)
        got = b.download_device(out).reshape(rows, stride)
        assert (got[:, n:] == 31).all()  # nothing beside the rows is written
        return got[:, :n]


SHAPES = [(1, 1, 1), (1, 64, 16), (1, 768, 2304), (2, 3, 5), (3, 65, 17), (7, 130, 50257), (15, 63, 15), (16, 64, 16),
          (17, 128, 33), (31, 200, 48), (33, 100, 50), (64, 192, 64), (65, 257, 70), (100, 70, 1000), (127, 64, 127),
          (128, 64, 128), (129, 65, 129), (300, 31, 300), (513, 130, 260), (1000, 16, 17), (2049, 77, 33)]


@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_linear_sums(backend, rows, k, n):
    g = gen(rows * 1000003 + k * 1009 + n)
    x, w = full(g, (rows, k)), full(g, (k, n))
    assert np.array_equal(run_linear(backend, x, w, raw=True), ref.linear(x, w, raw=True))


@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_linear_epilogue(backend, rows, k, n):
    g = gen(rows * 1000033 + k * 2003 + n)
    x, w = normal(g, (rows, k), 1000), normal(g, (k, n), 2000)
    kw = dict(bias=full(g, n), bias_shift=9, shift=int(np.log2(2e6 * np.sqrt(k) / 9000)), table=full(g, 65536),
              residual=full(g, (rows, n)))
    assert np.array_equal(run_linear(backend, x, w, **kw), ref.linear(x, w, **kw))


def check_linear_tiles(b, rows, k, n, large, seed=0):
    """Sums and an epilogue of every part, with weights (and x) over all of i16 or of ordinary size; the reference's sums
    are exact in doubles."""
    g = gen(rows + k + n + seed)
    x, w = (full(g, (rows, k)), full(g, (k, n))) if large else (normal(g, (rows, k), 1000), normal(g, (k, n), 2000))
    acc = ref._sums(x, w)
    shift = 31 if large else int(np.log2(2e6 * np.sqrt(k) / 9000))
    for s in (shift, min(shift, 11)):
        kw = dict(bias=full(g, n), bias_shift=9, shift=s, table=full(g, 65536), residual=full(g, (rows, n)))
        h = ref.sat(ref.rs(acc + kw["bias"].astype(np.int64) * 512, s))
        h = ref.sat(kw["table"].astype(np.int64)[h + 32768] + kw["residual"].astype(np.int64))
        assert np.array_equal(run_linear(b, x, w, **kw), h)
    assert np.array_equal(run_linear(b, x, w, raw=True, out_gap=3), acc)


@pytest.mark.parametrize("large", [False, True])
@pytest.mark.parametrize("rows,k,n", [
    (800, 136, 500), (801, 131, 497), (1500, 104, 1200), (1499, 99, 1201), (1600, 520, 2000), (1543, 509, 1990),
    (4090, 200, 2040), (4081, 199, 2033), (17, 64, 12000)])
def test_linear_of_many_rows_and_columns(backend, rows, k, n, large):
    """Tiles of every size, whole ones and those at the edges, with rows aligned and not."""
    check_linear_tiles(backend, rows, k, n, large)


def test_without_workspaces_in_a_coarse_scope():
    """Rows that are not aligned, and few rows of a long sequence, where no workspace may be allocated."""
    from volta_mi355x import Backend
    g = gen(77)
    x, w = normal(g, (801, 131), 1000), normal(g, (131, 497), 2000)
    q, k, v = normal(g, (1, 2, 64), 1000), normal(g, (3000, 2, 64), 1000), normal(g, (3000, 2, 64), 3000)
    with Backend(timing_policy=1) as b, Held(b) as held:
        dx, dq, table = held.put(x), held.put(q), held.put(exponentials())
        packed = b.fixed_weights_device(held.put(w), 131, 497)
        held.keep(packed.storage)
        cache = b.fixed_kv_cache(1, 2, 64, 3000)
        held.keep(cache.storage)
        b.fixed_kv_append_device(cache, held.put(k), held.put(v), [[0, 0, 3000, 3000]])
        y, o = held.new(801 * 497, np.int16), held.new(128, np.int16)
        live = b.get_stats()["live_device_bytes"]
        for run in (lambda: b.fixed_linear_device(dx, 801, packed, 12, out=y),
                    lambda: b.fixed_attention_device(dq, cache, [[0, 0, 1, 3000]], 2, table, 13, out=o)):
            assert b.lib.volta_cuda_begin_coarse_timing(b.raw, 0) == 0
            run()
            assert b.lib.volta_cuda_end_coarse_timing(b.raw) == 0
        assert b.get_stats()["live_device_bytes"] == live
        first = b.download_device(y).reshape(801, 497), b.download_device(o)
        b.fixed_linear_device(dx, 801, packed, 12, out=y)
        b.fixed_attention_device(dq, cache, [[0, 0, 1, 3000]], 2, table, 13, out=o)
        assert b.get_stats()["live_device_bytes"] > live
        second = b.download_device(y).reshape(801, 497), b.download_device(o)
    want = ref.sat(ref.rs(ref._sums(x, w), 12)), ref.attention(q, k, v, exponentials(), 13, True).reshape(-1)
    for got in (first, second):
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_attention_workspace_grows_in_few_steps():
    """A sequence that gets longer does not allocate again for every tile of tokens."""
    from volta_mi355x import Backend
    n = 6000
    g = gen(n)
    k, v, q = (normal(g, (m, 4, 64), s) for m, s in ((n, 1000), (n, 3000), (1, 1000)))
    with Backend(timing_policy=1) as b, Held(b) as held:
        cache = b.fixed_kv_cache(1, 4, 64, n)
        held.keep(cache.storage)
        b.fixed_kv_append_device(cache, held.put(k), held.put(v), [[0, 0, n, n]])
        dq, table, out = held.put(q), held.put(exponentials()), held.new(256, np.int16)
        before = b.get_stats()["allocation_calls"]
        for length in range(2100, n, 64):
            b.fixed_attention_device(dq, cache, [[0, 0, 1, length]], 4, table, 13, out=out)
            want = ref.attention(q, k[:length], v[:length], exponentials(), 13, True)
            assert np.array_equal(b.download_device(out).reshape(q.shape), want)
        assert 1 <= b.get_stats()["allocation_calls"] - before <= 3


def test_attention_workspace_is_bounded():
    """Scores of sequences whose space together would pass the bound (512 MiB) are taken some sequences at a time."""
    from volta_mi355x import Backend
    slots, kv_heads, heads, dim, n = 20, 8, 128, 16, 65536
    g = gen(5)
    k, v, q = (normal(g, (m, h, dim), s) for m, h, s in
               ((n, kv_heads, 1000), (n, kv_heads, 3000), (slots, heads, 1000)))
    with Backend(timing_policy=1) as b, Held(b) as held:
        cache = b.fixed_kv_cache(slots, kv_heads, dim, n)
        held.keep(cache.storage)
        dk, dv, dq, table = held.put(k), held.put(v), held.put(q), held.put(exponentials())
        lengths = [n - 1000 * i for i in range(slots)]
        b.fixed_kv_append_device(cache, dk, dv, [[i, 0, m, m] for i, m in enumerate(lengths)])
        out = held.new(q.size, np.int16)
        before = b.get_stats()["live_device_bytes"]
        b.fixed_attention_device(dq, cache, [[i, i, 1, m] for i, m in enumerate(lengths)], heads, table, 12, out=out)
        got = b.download_device(out).reshape(q.shape)
        assert 0 < b.get_stats()["live_device_bytes"] - before <= 512 << 20
    for i, m in enumerate(lengths):
        for kv in (i % 8, (i + 3) % 8):
            mine = slice(kv * 16, kv * 16 + 16)
            want = ref.attention(q[i:i + 1, mine], k[:m, kv:kv + 1], v[:m, kv:kv + 1], exponentials(), 12, True)
            assert np.array_equal(got[i:i + 1, mine], want), (i, kv)


@pytest.mark.parametrize("gap", [0, 3])
def test_linear_workspace_is_bounded(gap):
    """Rows that are not aligned are aligned some at a time (128 MiB)."""
    from volta_mi355x import Backend
    rows, k, n = 40000, 2001, 41
    g = gen(rows)
    wide, w = normal(g, (rows, k + gap), 1000), normal(g, (k, n), 2000)
    bias, table, res = full(g, n), full(g, 65536), full(g, (rows, n))
    acc = ref._sums(wide[:, :k], w)
    with Backend(timing_policy=1) as b, Held(b) as held:
        x, packed = held.put(wide), b.fixed_weights_device(held.put(w), k, n)
        held.keep(packed.storage)
        db, dt, dr = held.put(bias), held.put(table), held.put(res)
        y, sums = held.new(rows * (n + 2), np.int16, 7), held.new(rows * (n + 1), np.int64, 8)
        before = b.get_stats()["live_device_bytes"]
        b.fixed_linear_device(x, rows, packed, 14, x_stride=k + gap, bias=db, bias_shift=9, table=dt, residual=dr, out=y,
                              out_stride=n + 2)
        b.fixed_linear_device(x, rows, packed, x_stride=k + gap, raw=True, out=sums, out_stride=n + 1)
        y, sums = b.download_device(y).reshape(rows, -1), b.download_device(sums).reshape(rows, -1)
        assert 0 < b.get_stats()["live_device_bytes"] - before <= 128 << 20
    h = table.astype(np.int64)[ref.sat(ref.rs(acc + bias.astype(np.int64) * 512, 14)) + 32768]
    assert np.array_equal(y[:, :n], ref.sat(h + res)) and (y[:, n:] == 7).all()
    assert np.array_equal(sums[:, :n], acc) and (sums[:, n:] == 8).all()


@pytest.mark.parametrize("use", ["", "bias", "table", "residual", "bias table", "bias residual", "table residual"])
@pytest.mark.parametrize("rows,k,n", [(5, 100, 40), (200, 100, 150)])
def test_linear_optional_parts(backend, rows, k, n, use):
    g = gen(len(use) + rows)
    x, w = normal(g, (rows, k), 1000), normal(g, (k, n), 2000)
    kw = dict(shift=12)
    if "bias" in use:
        kw.update(bias=full(g, n), bias_shift=10)
    if "table" in use:
        kw["table"] = full(g, 65536)
    if "residual" in use:
        kw["residual"] = full(g, (rows, n))
    assert np.array_equal(run_linear(backend, x, w, **kw), ref.linear(x, w, **kw))


@pytest.mark.parametrize("rows", [4, 150])
@pytest.mark.parametrize("shift", [0, 1, 16, 17, 31, 32, 46, 62])
def test_linear_shifts_and_rounding(backend, rows, shift):
    g = gen(shift)
    x, w = full(g, (rows, 96)), full(g, (96, 40))
    kw = dict(shift=shift, bias=full(g, 40), bias_shift=46 if shift > 40 else 0)
    assert np.array_equal(run_linear(backend, x, w, **kw), ref.linear(x, w, **kw))


@pytest.mark.parametrize("rows", [1, 20, 140])
@pytest.mark.parametrize("gap,offset", [(0, 1), (1, 0), (3, 5), (8, 8), (13, 2)])
def test_linear_strides_and_alignment(backend, rows, gap, offset):
    g = gen(gap * 10 + offset)
    x, w, res = full(g, (rows, 77)), full(g, (77, 35)), full(g, (rows, 35))
    kw = dict(shift=20, residual=res)
    got = run_linear(backend, x, w, x_gap=gap, x_offset=offset, out_gap=gap + 1, residual_gap=gap, **kw)
    assert np.array_equal(got, ref.linear(x, w, **kw))


@pytest.mark.parametrize("rows", [1, 129])
@pytest.mark.parametrize("a,b_", [(-32768, -32768), (-32768, 32767), (32767, 32767), (127, -129)])
def test_linear_longest_sums_of_equal_values(backend, rows, a, b_):
    """k = 65,535 equal products: the i32 partial sums at their ends."""
    k = 65535
    x, w = np.full((rows, k), a, np.int16), np.full((k, 3), b_, np.int16)
    got = run_linear(backend, x, w, raw=True)
    assert (got == k * a * b_).all()


@pytest.mark.parametrize("rows", [3, 70, 200])
@pytest.mark.parametrize("top", [32639, 32640, 32767])
@pytest.mark.parametrize("cols", [[0], [37], [149], [16, 17, 140]])
def test_linear_few_large_weights(backend, rows, top, cols):
    """Columns whose weights need the offset of their low byte beside columns that do not."""
    g = gen(top + rows)
    x, w = full(g, (rows, 130)), normal(g, (130, 150), 2000)
    for c in cols:
        w[g.integers(0, 130), c] = top
    kw = dict(shift=13, bias=full(g, 150), bias_shift=11)
    assert np.array_equal(run_linear(backend, x, w, raw=True), ref.linear(x, w, raw=True))
    assert np.array_equal(run_linear(backend, x, w, **kw), ref.linear(x, w, **kw))


@pytest.mark.parametrize("rows", [2, 100])
def test_linear_offset_beside_the_longest_column(backend, rows):
    """One large weight gives its 16 columns the offset; another of them is -32,768 throughout (its offset
    values sum to less than -2^31)."""
    k = 65535
    w = np.full((k, 3), -32768, np.int16)
    w[5, 0] = 32767
    x = np.full((rows, k), 3, np.int16)
    x[0] = -32768
    want = np.stack([x[:, 0].astype(np.int64) * int(w[:, c].astype(np.int64).sum()) for c in range(3)], 1)
    assert np.array_equal(run_linear(backend, x, w, raw=True), want)


def test_linear_transposed_weights_and_stride(backend):
    g = gen(3)
    x, w = full(g, (9, 70)), full(g, (70, 41))
    assert np.array_equal(run_linear(backend, x, w, transposed=True, raw=True), ref.linear(x, w, raw=True))
    with Held(backend) as held:  # a tensor inside a wider commitment block
        wide = np.full((70, 64), 999, np.int16)
        wide[:, 5:46] = w
        dw, dx = held.put(wide), held.put(x)
        packed = backend.fixed_weights_device(dw, 70, 41, offset=5, stride=64)
        held.keep(packed.storage)
        out = held.keep(backend.fixed_linear_device(dx, 9, packed, raw=True))
        assert np.array_equal(backend.download_device(out).reshape(9, 41), ref.linear(x, w, raw=True))


@pytest.mark.parametrize("rows", [6, 300])
def test_linear_over_its_residual(backend, rows):
    g = gen(rows)
    x, w, res = normal(g, (rows, 64), 1000), normal(g, (64, 50), 2000), full(g, (rows, 50))
    with Held(backend) as held:
        dx, dr = held.put(x), held.put(res)
        packed = backend.fixed_weights_device(held.put(w), 64, 50)
        held.keep(packed.storage)
        backend.fixed_linear_device(dx, rows, packed, 10, residual=dr, out=dr)
        assert np.array_equal(backend.download_device(dr).reshape(rows, 50), ref.linear(x, w, shift=10, residual=res))


# ---- attention ------------------------------------------------------------------------------

def run_attention(b, q, k, v, lengths, counts, past, table, shift, *, causal=True, capacity=None, gap=0, slots=None,
                  q_offset=0):
    """Packed rows of several sequences; past[i]: their earlier (keys, values)."""
    heads, dim, kv_heads = q.shape[1], q.shape[2], k.shape[1]
    with Held(b) as held:
        capacity = capacity or max(max(lengths), 1)
        order = list(range(len(lengths))) if slots is None else slots
        cache = b.fixed_kv_cache(max(order) + 1, kv_heads, dim, capacity)
        held.keep(cache.storage)
        # garbage in every byte first: places that no token fills must not matter
        b.upload_into(cache.storage, 0, gen(9).integers(0, 256, min(cache.storage.len, 1 << 26), dtype=np.uint8))
        first = np.concatenate([[0], np.cumsum(counts)[:-1]]).astype(np.int64)
        for i, (pk, pv) in enumerate(past):
            if len(pk):
                b.fixed_kv_append_device(cache, held.put(pk), held.put(pv), [[order[i], 0, len(pk), len(pk)]])

        def wide(a):
            flat = a.reshape(len(a), -1)
            w = np.full((len(a), flat.shape[1] + gap), -3333, np.int16)
            w[:, :flat.shape[1]] = flat
            return held.put(np.concatenate([np.full(q_offset, 5, np.int16), w.reshape(-1)]))

        cols, kv_cols = heads * dim, kv_heads * dim
        news = np.minimum(counts, lengths)
        if (np.array(counts) <= np.array(lengths)).all():
            seqs = np.stack([order, first, counts, lengths], 1)
            b.fixed_kv_append_device(cache, wide(k), wide(v), seqs, k_offset=q_offset, k_stride=kv_cols + gap,
                                     v_offset=q_offset, v_stride=kv_cols + gap)
        else:
            assert not causal and not news.any()
            seqs = np.stack([order, first, counts, lengths], 1)
        out = held.new(len(q) * (cols + gap) + q_offset, np.int16, 99)
        b.fixed_attention_device(wide(q), cache, seqs, heads, held.put(table), shift, causal=causal, q_offset=q_offset,
                                 q_stride=cols + gap, out=out, out_offset=q_offset, out_stride=cols + gap)
        got = b.download_device(out)
        assert (got[:q_offset] == 99).all()
        got = got[q_offset:].reshape(len(q), cols + gap)
        assert (got[:, cols:] == 99).all()
        return got[:, :cols].reshape(q.shape)


def attention_case(seed, counts, lengths, heads, kv_heads, dim, std=1000, values=3000):
    g = gen(seed)
    rows = sum(counts)
    make = (lambda s: full(g, s)) if std is None else (lambda s: normal(g, s, std))
    q, k = make((rows, heads, dim)), make((rows, kv_heads, dim))
    v = full(g, (rows, kv_heads, dim)) if values is None else normal(g, (rows, kv_heads, dim), values)
    past = []
    for c, n in zip(counts, lengths):
        p = max(0, n - c)
        past.append((make((p, kv_heads, dim)),
                     full(g, (p, kv_heads, dim)) if values is None else normal(g, (p, kv_heads, dim), values)))
    return q, k, v, past


def want_attention(q, k, v, lengths, counts, past, table, shift, causal=True):
    out, at = np.zeros(q.shape, np.int16), 0
    for c, n, (pk, pv) in zip(counts, lengths, past):
        keys, vals = (np.concatenate([p, t[at:at + c]])[:n] for p, t in ((pk, k), (pv, v)))
        out[at:at + c] = ref.attention(q[at:at + c], keys, vals, table, shift, causal)
        at += c
    return out


def check_attention(b, seed, counts, lengths, heads, kv_heads, dim, *, table=None, shift=None, causal=True, std=1000,
                    values=3000, **kw):
    table = exponentials() if table is None else table
    shift = max(8, round(np.log2(np.sqrt(dim) * 1e6 / 1280))) if shift is None else shift
    q, k, v, past = attention_case(seed, counts, lengths, heads, kv_heads, dim, std, values)
    got = run_attention(b, q, k, v, lengths, counts, past, table, shift, causal=causal, **kw)
    want = want_attention(q, k, v, lengths, counts, past, table, shift, causal)
    bad = np.argwhere(got != want)
    assert not len(bad), (len(bad), bad[:4].tolist())


@pytest.mark.parametrize("dim", [1, 15, 16, 40, 63, 64, 65, 80, 96, 127, 128])
@pytest.mark.parametrize("counts,lengths", [([1], [1]), ([3, 70], [3, 70]), ([1, 1, 5], [64, 65, 200])])
def test_attention_head_sizes(backend, dim, counts, lengths):
    check_attention(backend, dim, counts, lengths, 4, 2, dim)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (12, 12), (8, 2), (20, 1), (6, 3), (40, 2), (70, 1)])
@pytest.mark.parametrize("counts,lengths", [([1, 1], [130, 63]), ([2, 40, 129], [2, 100, 129])])
def test_attention_grouped_heads(backend, heads, kv_heads, counts, lengths):
    check_attention(backend, heads * 100 + kv_heads, counts, lengths, heads, kv_heads, 64)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 320])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_prompt_lengths(backend, n, dim):
    check_attention(backend, n, [n, 5], [n, 5], 2, 1, dim)


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 128, 129, 1000, 1024, 4095, 4097, 9000])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 4])
def test_attention_tokens_over_a_cache(backend, n, dim, new):
    n = max(n, new)
    check_attention(backend, n + new, [new, 1, new], [n, max(1, n // 3), max(new, n - 1)], 4, 2, dim)


@pytest.mark.parametrize("batch,longest,heads,kv_heads,dim", [
    (40, 300, 16, 8, 64), (9, 1300, 12, 12, 64), (2, 1300, 2, 2, 64), (9, 1300, 12, 12, 128), (70, 3300, 2, 1, 64),
    (130, 700, 3, 1, 80)])
def test_attention_tokens_of_many_sequences(backend, batch, longest, heads, kv_heads, dim):
    """Few and many sequences a launch, and several launches, with lengths from one token to the longest."""
    lengths = [max(1, longest * ((7 * i) % 11) // 11) if i else longest for i in range(batch)]
    check_attention(backend, batch, [1] * batch, lengths, heads, kv_heads, dim)


@pytest.mark.parametrize("new", [17, 40, 100, 200])
def test_attention_prompts_in_pieces(backend, new):
    check_attention(backend, new, [new, 1, new + 3], [new + 700, 333, new + 64], 4, 1, 64)


@pytest.mark.parametrize("causal", [True, False])
def test_attention_without_the_causal_mask(backend, causal):
    check_attention(backend, 5, [70, 1, 3], [70, 300, 90], 2, 2, 64, causal=causal)


def test_attention_rows_that_see_nothing_are_zero(backend):
    """Empty slots under no causal mask, beside sequences that have tokens."""
    g = gen(4)
    q = normal(g, (9, 2, 64), 1000)
    with Held(backend) as held:
        cache = backend.fixed_kv_cache(3, 2, 64, 100)
        held.keep(cache.storage)
        backend.upload_into(cache.storage, 0, g.integers(0, 256, cache.storage.len, dtype=np.uint8))
        k, v = normal(g, (4, 2, 64), 1000), normal(g, (4, 2, 64), 3000)
        backend.fixed_kv_append_device(cache, held.put(k), held.put(v), [[1, 0, 4, 4]])
        out = held.new(9 * 128, np.int16, 7)
        backend.fixed_attention_device(held.put(q), cache, [[0, 0, 3, 0], [1, 3, 5, 4], [2, 8, 1, 0]], 2,
                                       held.put(exponentials()), 13, causal=False, out=out)
        got = backend.download_device(out).reshape(q.shape)
    assert not got[:3].any() and not got[8:].any()
    assert np.array_equal(got[3:8], ref.attention(q[3:8], k, v, exponentials(), 13, False))


@pytest.mark.parametrize("shift", [8, 9, 15, 16, 17, 20, 24])
@pytest.mark.parametrize("counts,lengths", [([1, 2], [200, 70]), ([90], [90])])
def test_attention_shifts_with_values_at_the_ends(backend, shift, counts, lengths):
    """Queries, keys and values over all of i16: scores up to 2^37."""
    for dim in (64, 128):
        check_attention(backend, shift, counts, lengths, 2, 1, dim, shift=shift, std=None, values=None,
                        table=exponentials(ENTRIES, 40.0 * 2 ** (24 - shift) / 16))


@pytest.mark.parametrize("entries", [1, 2, 5, 1000, 8192])
def test_attention_table_lengths(backend, entries):
    g = gen(entries)
    table = g.integers(0, 16385, entries).astype(np.uint16)
    check_attention(backend, entries, [1, 40], [100, 60], 2, 1, 64, table=table)


def test_attention_table_beyond_its_range_and_all_zero(backend):
    big = np.full(100, 60000, np.uint16)
    big[::3] = 16385
    big[::7] = 3
    check_attention(backend, 1, [1, 40], [100, 60], 2, 1, 64, table=big)
    check_attention(backend, 1, [1, 40], [100, 60], 2, 1, 64, table=np.zeros(50, np.uint16))


@pytest.mark.parametrize("gap,offset", [(0, 1), (1, 0), (7, 3), (64, 8)])
def test_attention_strides_and_alignment(backend, gap, offset):
    check_attention(backend, gap, [1, 33], [70, 33], 4, 2, 40, gap=gap, q_offset=offset)
    check_attention(backend, gap, [130, 2], [130, 5], 4, 4, 64, gap=gap, q_offset=offset)


def test_attention_many_sequences(backend):
    g = gen(11)
    counts = [int(x) for x in g.integers(0, 4, 150)]
    lengths = [c + int(x) for c, x in zip(counts, g.integers(0, 90, 150))]
    check_attention(backend, 12, counts, lengths, 2, 1, 64, slots=[int(x) for x in g.permutation(150)])
    counts = [int(x) for x in g.integers(0, 60, 70)]
    check_attention(backend, 13, counts, [c + 7 for c in counts], 6, 2, 64)


def prompts(g, batch, longest, past=0):
    """Sequences enough to fill the GPU with 128-row pieces: one of the longest, the rest of any length."""
    counts = [longest] + [int(x) for x in g.integers(1, longest + 1, batch - 1)]
    return counts, [c + (int(g.integers(0, past + 1)) if past else 0) for c in counts]


@pytest.mark.parametrize("batch,heads,kv_heads", [(5, 12, 12), (20, 12, 12), (9, 32, 8)])
@pytest.mark.parametrize("dim", [33, 64, 100, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_many_prompts(backend, batch, heads, kv_heads, dim, causal):
    g = gen(batch * 1000 + dim + causal)
    counts, lengths = prompts(g, batch, 300)
    check_attention(backend, dim, counts, lengths, heads, kv_heads, dim, causal=causal)


@pytest.mark.parametrize("batch", [6, 20])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_many_prompts_over_a_past(backend, batch, dim):
    counts, lengths = prompts(gen(batch + dim), batch, 260, past=150)
    check_attention(backend, dim, counts, lengths, 12, 12, dim, gap=9, q_offset=3)


@pytest.mark.parametrize("batch", [6, 20])
@pytest.mark.parametrize("dim", [64, 127])
@pytest.mark.parametrize("shift", [8, 16, 17, 24])
def test_attention_many_prompts_with_values_at_the_ends(backend, batch, dim, shift):
    counts, lengths = prompts(gen(batch + dim), batch, 150, past=40)
    check_attention(backend, shift, counts, lengths, 24, 24, dim, shift=shift, std=None, values=None,
                    table=exponentials(ENTRIES - 3, 40.0 * 2 ** (24 - shift) / 16))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("key", [32639, 32640])
def test_attention_few_large_keys_and_queries(backend, dim, key):
    """Tokens that need the offset of their low byte beside tokens that do not, in both kernels."""
    for counts, lengths in (([1, 3], [200, 70]), prompts(gen(dim), 20, 200)):
        g = gen(key)
        q, k, v, past = attention_case(3, counts, lengths, 12, 12, dim)
        for t in [q, k] + [p for p, _ in past if len(p)]:
            flat = t.reshape(-1)
            flat[g.integers(0, flat.size, max(1, flat.size // 4000))] = key
        shift = max(8, round(np.log2(np.sqrt(dim) * 1e6 / 1280))) + 3
        got = run_attention(backend, q, k, v, lengths, counts, past, exponentials(), shift)
        assert np.array_equal(got, want_attention(q, k, v, lengths, counts, past, exponentials(), shift))


def test_attention_appends_in_pieces(backend):
    """Tokens written one to three at a time, at every place of a tile, leave the same cache as one append."""
    g = gen(21)
    q, k, v = (normal(g, (150, 2, 80), s) for s in (1000, 1000, 3000))
    table, want = exponentials(), None
    with Held(backend) as held:
        dq, dk, dv, dt = held.put(q), held.put(k), held.put(v), held.put(table)
        for pieces in ([150], [1] * 150, [3, 2] * 30, [63, 1, 1, 85], [64, 64, 22]):
            cache = backend.fixed_kv_cache(2, 2, 80, 160)
            at = 0
            for p in pieces:
                backend.fixed_kv_append_device(cache, dk, dv, [[1, at, p, at + p]])
                at += p
            out = backend.fixed_attention_device(dq, cache, [[1, 0, 150, 150]], 2, dt, 14)
            got = backend.download_device(out)
            backend.free_device(out)
            backend.free_fixed_kv_cache(cache)
            want = ref.attention(q, k, v, table, 14, True).reshape(-1) if want is None else want
            assert np.array_equal(got, want), pieces


@pytest.mark.parametrize("dim", [40, 64, 128])
def test_append_writes_only_its_own_places(backend, dim):
    """Tokens written again leave those after them in their tile as they were."""
    g = gen(dim)
    n = 200
    q, k, v = (normal(g, (n, 2, dim), s) for s in (1000, 1000, 3000))
    table = exponentials()
    with Held(backend) as held:
        cache = backend.fixed_kv_cache(2, 2, dim, 230)
        held.keep(cache.storage)
        backend.upload_into(cache.storage, 0, g.integers(0, 256, cache.storage.len, dtype=np.uint8))
        backend.fixed_kv_append_device(cache, held.put(k), held.put(v), [[1, 0, n, n]])
        dq, dt, out = held.put(q), held.put(table), held.new(n * 2 * dim, np.int16)
        for first, count in ((0, 10), (0, 1), (64, 3), (128, 63), (60, 10), (0, 100), (5, 5), (192, 5), (64, 64), (0, 29),
                             (64, 36)):
            k[first:first + count] = full(g, (count, 2, dim))
            v[first:first + count] = full(g, (count, 2, dim))
            backend.fixed_kv_append_device(cache, held.put(k[first:first + count]), held.put(v[first:first + count]),
                                           [[1, 0, count, first + count]])
            backend.fixed_attention_device(dq, cache, [[1, 0, n, n]], 2, dt, 16, out=out)
            assert np.array_equal(backend.download_device(out).reshape(q.shape), ref.attention(q, k, v, table, 16, True)), (
                first, count)


@pytest.mark.parametrize("new", [1, 3])
@pytest.mark.parametrize("value,e", [(-32768, 16384), (32767, 16384), (-32768, 129), (255, 128)])
def test_attention_longest_sums_of_equal_values(backend, new, value, e):
    """65,536 equal keys and values: the i32 partial sums at their ends."""
    n = 65536
    with Held(backend) as held:
        cache = backend.fixed_kv_cache(1, 1, 64, n)
        held.keep(cache.storage)
        same = held.put(np.full((n, 64), value, np.int16))
        backend.fixed_kv_append_device(cache, same, same, [[0, 0, n, n]])
        q = held.put(np.full((new, 64), -32768, np.int16))
        out = held.keep(backend.fixed_attention_device(q, cache, [[0, 0, new, n]], 1,
                                                       held.put(np.full(3, e, np.uint16)), 8))
        assert (backend.download_device(out) == value).all()


def test_attention_cache_records_past_four_gib(backend):
    """Slots whose records start beyond 2^32 bytes."""
    slots, heads, n = 300, 2, 32768
    with Held(backend) as held:
        cache = backend.fixed_kv_cache(slots, heads, 64, n)
        held.keep(cache.storage)
        assert cache.storage.nbytes > 4 << 30
        g = gen(8)
        k, v, q = (normal(g, (100, heads, 64), s) for s in (1000, 3000, 1000))
        backend.fixed_kv_append_device(cache, held.put(k), held.put(v), [[slots - 1, 0, 50, 50], [0, 50, 50, 50]])
        out = held.keep(backend.fixed_attention_device(held.put(q), cache, [[slots - 1, 0, 50, 50], [0, 50, 50, 50]],
                                                       heads, held.put(exponentials()), 13))
        got = backend.download_device(out).reshape(100, heads, 64)
    for part in (slice(0, 50), slice(50, 100)):
        assert np.array_equal(got[part], ref.attention(q[part], k[part], v[part], exponentials(), 13, True))


@pytest.mark.parametrize("policy", [0, 1])
@pytest.mark.parametrize("kv_heads,length", [(1, 200), (1, 600), (2, 4000)])
def test_attention_reports_a_failed_launch(policy, kv_heads, length):
    """The check after a launch reads this thread's last HIP error, so an error left by a call before it takes
    the way of a launch that fails: the call says so and runs no other kernel in its place."""
    from volta_mi355x import Backend, GpuError
    g = gen(length)
    q, k, v = (normal(g, (n, kv_heads, 64), s) for n, s in ((1, 1000), (length, 1000), (length, 3000)))
    with Backend(timing_policy=policy) as b, Held(b) as held:
        cache = b.fixed_kv_cache(1, kv_heads, 64, length)
        held.keep(cache.storage)
        b.fixed_kv_append_device(cache, held.put(k), held.put(v), [[0, 0, length, length]])
        dq, table, out = held.put(q), held.put(exponentials()), held.new(kv_heads * 64, np.int16)

        def attend():
            return b.fixed_attention_device(dq, cache, [[0, 0, 1, length]], kv_heads, table, 13, out=out)

        attend()
        b.synchronize()
        assert b.lib.hipSetDevice(1 << 20) != 0
        with pytest.raises(GpuError, match="hipGetLastError"):
            attend()
        attend()
        assert np.array_equal(b.download_device(out).reshape(q.shape),
                              ref.attention(q, k, v, exponentials(), 13, True))


# ---- rows -----------------------------------------------------------------------------------

@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 2), (3, 7), (2, 64), (5, 65), (4, 255), (3, 256), (9, 768),
                                       (2, 1000), (3, 1025), (2, 2048), (2, 4095), (2, 8192), (1, 8193), (1, 20000),
                                       (1, 65536), (700, 33)])
def test_norm(backend, rows, cols, residual, rms):
    g = gen(rows * 70001 + cols)
    b = backend
    for spread in (30, 30000):
        x, res = normal(g, (rows, cols), spread), normal(g, (rows, cols), 2 * spread) if residual else None
        gain, bias = full(g, cols), full(g, cols) if cols % 2 else None
        for shift, eps in ((0, 1), (2, cols * cols), (15, 1 << 40)):
            with Held(b) as held:
                kept = held.new(rows * (cols + 3), np.int16, 5)
                out = held.new(rows * (cols + 1), np.int16, 6)
                b.fixed_norm_device(held.put(x), rows, cols, held.put(gain), shift, eps, bias=held.put(bias),
                                    rms=rms, residual=held.put(res), sum_out=kept, sum_stride=cols + 3, out=out,
                                    out_stride=cols + 1)
                y, h = (b.download_device(t).reshape(rows, -1) for t in (out, kept))
            want, want_h = ref.norm(x, gain, shift, eps, bias=bias, residual=res, rms=rms)
            assert np.array_equal(y[:, :cols], want) and (y[:, cols:] == 6).all()
            assert np.array_equal(h[:, :cols], want_h) and (h[:, cols:] == 5).all()


@pytest.mark.parametrize("cols", [512, 513, 1024, 1500, 2049, 4096, 4097])
def test_norm_widths(backend, cols):
    g = gen(cols)
    x, gain, bias = normal(g, (5, cols), 3000), full(g, cols), full(g, cols)
    with Held(backend) as held:
        out = held.keep(backend.fixed_norm_device(held.put(x), 5, cols, held.put(gain), 3, cols, bias=held.put(bias)))
        got = backend.download_device(out).reshape(5, cols)
    assert np.array_equal(got, ref.norm(x, gain, 3, cols, bias=bias)[0])


@pytest.mark.parametrize("cols", [2, 768, 65536])
def test_norm_of_values_at_the_ends(backend, cols):
    rows = np.stack([np.full(cols, -32768), np.full(cols, 32767), np.where(np.arange(cols) % 2, -32768, 32767),
                     np.zeros(cols), np.arange(cols) == 0]).astype(np.int16)
    gain = np.full(cols, -32768, np.int16)
    gain[::3] = 32767
    for rms in (False, True):
        for eps in (1, 1 << 40):
            with Held(backend) as held:
                out = held.keep(backend.fixed_norm_device(held.put(rows), 5, cols, held.put(gain), 0, eps, rms=rms))
                got = backend.download_device(out).reshape(5, cols)
            assert np.array_equal(got, ref.norm(rows, gain, 0, eps, rms=rms)[0])


@pytest.mark.parametrize("cols", [64, 777, 9000])
def test_norm_sum_over_x_or_over_the_residual(backend, cols):
    g = gen(cols)
    x, res, gain = full(g, (3, cols)), full(g, (3, cols)), normal(g, cols, 4000)
    want, h = ref.norm(x, gain, 3, 5, residual=res)
    for over in (0, 1):
        with Held(backend) as held:
            t = [held.put(x), held.put(res)]
            out = held.keep(backend.fixed_norm_device(t[0], 3, cols, held.put(gain), 3, 5, residual=t[1],
                                                      sum_out=t[over]))
            assert np.array_equal(backend.download_device(out).reshape(3, cols), want)
            assert np.array_equal(backend.download_device(t[over]).reshape(3, cols), h)


@pytest.mark.parametrize("rows,cols,vocab", [(1, 1, 1), (1, 768, 50), (5, 7, 3), (33, 64, 9), (200, 769, 40), (3, 5000, 4)])
@pytest.mark.parametrize("places", [False, True])
def test_embed(backend, rows, cols, vocab, places):
    g = gen(rows * 1000 + cols)
    table, where = full(g, (vocab, cols)), full(g, (6, cols))
    tokens = g.integers(-2, vocab + 2, rows).astype(np.int32)
    tokens[0] = vocab - 1
    if rows > 3:
        tokens[1], tokens[2] = -(1 << 31), (1 << 31) - 1
    at = g.integers(-1, 8, rows).astype(np.int32) if places else None
    for scale, shift in ((1, 0), (23170, 14), (-(1 << 31), 46), ((1 << 31) - 1, 20)):
        with Held(backend) as held:
            out = held.new(rows * (cols + 2), np.int16, 4)
            kw = dict(positions=held.put(at), position_table=held.put(where), position_rows=6) if places else {}
            backend.fixed_embed_device(held.put(tokens), rows, held.put(table), vocab, cols, scale=scale, shift=shift,
                                       out=out, out_stride=cols + 2, **kw)
            got = backend.download_device(out).reshape(rows, cols + 2)
        want = ref.embed(tokens, table, scale=scale, shift=shift, positions=at, position_table=where if places else None)
        assert np.array_equal(got[:, :cols], want) and (got[:, cols:] == 4).all()


# ---- use and refusals -------------------------------------------------------------------------

def test_operators_are_counted_and_run_in_two_contexts():
    from volta_mi355x import Backend
    g = gen(2)
    x, w = full(g, (40, 64)), full(g, (64, 30))
    with Backend(timing_policy=1) as a, Backend() as b:
        jobs = []
        for ctx in (a, b, a, b):
            ctx.reset_stats()
            packed = ctx.fixed_weights_device(ctx.upload_device(w), 64, 30)
            jobs.append((ctx, ctx.fixed_linear_device(ctx.upload_device(x), 40, packed, raw=True)))
            assert ctx.get_stats()["calls"]["gemm"] == 2
        for ctx, out in jobs:
            assert np.array_equal(ctx.download_device(out).reshape(40, 30), ref.linear(x, w, raw=True))


def test_refusals(backend):
    from volta_mi355x import GpuError, InvalidInput
    b = backend
    with Held(b) as held:
        x, w = held.new(4096, np.int16), held.new(4096, np.int16)
        i32, i64 = held.new(64, np.int32), held.new(64, np.int64)
        table, exp = held.new(65536, np.int16), held.put(exponentials())
        packed = b.fixed_weights_device(w, 64, 32)
        held.keep(packed.storage)
        cache = b.fixed_kv_cache(2, 2, 16, 70)
        held.keep(cache.storage)
        refused = [
            lambda: b.fixed_weights_device(w, 65536, 1),
            lambda: b.fixed_weights_device(w, 0, 4),
            lambda: b.fixed_weights_device(w, 65, 64),
            lambda: b.fixed_weights_device(w, 64, 32, stride=31),
            lambda: b.fixed_weights_device(i32, 8, 8),
            lambda: b.fixed_linear_device(x, 0, packed, 4),
            lambda: b.fixed_linear_device(x, 65, packed, 4),
            lambda: b.fixed_linear_device(x, 4, packed, 63),
            lambda: b.fixed_linear_device(x, 4, packed, -1),
            lambda: b.fixed_linear_device(x, 4, packed, 4, bias_shift=47),
            lambda: b.fixed_linear_device(x, 4, packed, 4, x_stride=63),
            lambda: b.fixed_linear_device(x, 4, packed, 4, x_offset=4000),
            lambda: b.fixed_linear_device(x, 4, packed, raw=True, residual=w),
            lambda: b.fixed_linear_device(x, 4, packed, raw=True, table=table),
            lambda: b.fixed_linear_device(x, 4, packed, 4, table=w),
            lambda: b.fixed_linear_device(x, 4, packed, 4, out=i64),
            lambda: b.fixed_linear_device(x, 4, packed, 4, out=x),             # overlaps x
            lambda: b.fixed_linear_device(x, 4, packed, 4, residual=w, out=w, out_offset=1),
            lambda: b.fixed_kv_cache(1, 1, 129, 10),
            lambda: b.fixed_kv_cache(1, 1, 64, 65537),
            lambda: b.fixed_kv_cache(0, 1, 64, 10),
            lambda: b.fixed_kv_append_device(cache, x, w, [[2, 0, 1, 1]]),     # slot
            lambda: b.fixed_kv_append_device(cache, x, w, [[0, 0, 1, 71]]),    # capacity
            lambda: b.fixed_kv_append_device(cache, x, w, [[0, 0, 2, 1]]),     # more rows than tokens
            lambda: b.fixed_kv_append_device(cache, x, w, [[0, 0, 1, 1], [0, 1, 1, 2]]),
            lambda: b.fixed_kv_append_device(cache, x, w, [[0, 200, 1, 1]]),   # rows of k
            lambda: b.fixed_kv_append_device(cache, x, w, [[0, -1, 1, 1]]),
            lambda: b.fixed_attention_device(x, cache, [[0, 0, 1, 1]], 3, exp, 12),
            lambda: b.fixed_attention_device(x, cache, [[0, 0, 1, 1]], 2, exp, 7),
            lambda: b.fixed_attention_device(x, cache, [[0, 0, 1, 1]], 2, exp, 25),
            lambda: b.fixed_attention_device(x, cache, [[0, 0, 1, 1]], 2, table, 12),  # too many entries
            lambda: b.fixed_attention_device(x, cache, [[0, 0, 1, 1]], 2, i32, 12),
            lambda: b.fixed_attention_device(x, cache, [[0, 0, 2, 1]], 2, exp, 12),    # causal
            lambda: b.fixed_attention_device(x, cache, [[0, 0, 2, 5], [1, 1, 1, 5]], 2, exp, 12),
            lambda: b.fixed_attention_device(x, cache, [[0, 0, 1, 71]], 2, exp, 12),
            lambda: b.fixed_attention_device(x, cache, [[0, 0, 1, 1]], 2, exp, 12, out=x),
            lambda: b.fixed_attention_device(x, cache, [[0, 0, 200, 70]], 2, exp, 12, causal=False),
            lambda: b.fixed_norm_device(x, 2, 65537, w, 0, 1),
            lambda: b.fixed_norm_device(x, 2, 64, w, 16, 1),
            lambda: b.fixed_norm_device(x, 2, 64, w, 0, 0),
            lambda: b.fixed_norm_device(x, 2, 64, w, 0, (1 << 40) + 1),
            lambda: b.fixed_norm_device(x, 100, 64, w, 0, 1),
            lambda: b.fixed_norm_device(x, 2, 64, w, 0, 1, out=x),
            lambda: b.fixed_norm_device(x, 2, 64, w, 0, 1, sum_out=x, sum_offset=1),
            lambda: b.fixed_norm_device(x, 2, 64, i32, 0, 1),
            lambda: b.fixed_embed_device(i32, 65, w, 10, 16),
            lambda: b.fixed_embed_device(i32, 4, w, 1000, 16),
            lambda: b.fixed_embed_device(x, 4, w, 10, 16),
            lambda: b.fixed_embed_device(i32, 4, w, 10, 16, shift=47),
            lambda: b.fixed_embed_device(i32, 4, w, 10, 16, positions=i32),
            lambda: b.fixed_embed_device(i32, 4, w, 10, 16, out=w),
        ]
        for i, call in enumerate(refused):
            try:
                call()
            except (InvalidInput, GpuError):
                continue
            pytest.fail(f"call {i} was not refused")
        # the context works as before
        out = held.keep(b.fixed_linear_device(x, 4, packed, 4))
        assert not b.download_device(out).any()


@pytest.mark.parametrize("sequences", [[[0, 0, 1.5, 2]], np.array([[0.0, 0.0, 1.0, 1.0]]), [[0, 0], [1, 1]],
                                       np.zeros((4, 8), np.int64), [0, 0, 1], [[0, 0, 1, 1], [1, 1]], [["0", "0", "1", "1"]]])
def test_sequences_are_rows_of_four_integers(backend, sequences):
    from volta_mi355x import InvalidInput
    b = backend
    with Held(b) as held:
        x, w, exp, out = (held.new(4096, np.int16) for _ in range(4))
        cache = b.fixed_kv_cache(2, 2, 16, 70)
        held.keep(cache.storage)
        with pytest.raises(InvalidInput):
            b.fixed_kv_append_device(cache, x, w, sequences)
        with pytest.raises(InvalidInput):
            b.fixed_attention_device(x, cache, sequences, 2, exp, 12, out=out)
        for none in ([], np.zeros((0, 4), np.int64)):
            b.fixed_kv_append_device(cache, x, w, none)
            b.fixed_attention_device(x, cache, none, 2, exp, 12, out=out)


def test_refusals_at_the_c_entry(backend):
    """Arguments that the Python layer would catch first, straight through the ABI."""
    import ctypes

    from volta_mi355x import accel
    b, lib = backend, backend.lib
    with Held(b) as held:
        x = held.new(256, np.int16)
        packed = b.fixed_weights_device(x, 16, 16)
        held.keep(packed.storage)

        def linear(**kw):
            a = accel._FixedLinear(x_id=x.id, x_stride=16, weights_id=packed.storage.id, out_id=held.new(256, np.int16).id,
                                   out_stride=16, rows=4, k=16, n=16)
            for name, value in kw.items():
                setattr(a, name, value)
            return lib.volta_mi355x_fixed_linear_device(b.raw, ctypes.byref(a))

        assert linear() == 0
        for kw in (dict(x_id=0), dict(x_id=999), dict(x_stride=15), dict(rows=0), dict(rows=17), dict(rows=1 << 63),
                   dict(k=0), dict(k=1 << 40), dict(n=1 << 60), dict(x_off=1 << 63), dict(x_stride=1 << 62),
                   dict(shift=63), dict(bias_shift=47), dict(weights_off_bytes=8), dict(weights_id=0),
                   dict(out_id=packed.storage.id), dict(out_stride=15), dict(residual_id=x.id)):
            assert linear(**kw) != 0, kw
            assert b.last_error(), kw
        assert linear() == 0
        c = accel._FixedCache(x.id, 0, 1, 1, 64, 1 << 20)
        s = np.zeros((1, 4), np.int64)
        assert lib.volta_mi355x_fixed_kv_append_device(b.raw, ctypes.byref(c), x.id, 0, 64, x.id, 0, 64, s.ctypes.data, 1)
        c = accel._FixedCache(x.id, 0, 1, 1, 64, 64)  # the buffer is too short for its records
        assert lib.volta_mi355x_fixed_kv_append_device(b.raw, ctypes.byref(c), x.id, 0, 64, x.id, 0, 64, s.ctypes.data, 1)
        assert lib.volta_mi355x_fixed_kv_append_device(b.raw, None, x.id, 0, 64, x.id, 0, 64, s.ctypes.data, 1)
        for name in ("linear", "attention", "norm", "embed"):
            args = [None, None, 0] if name == "attention" else []
            fn = getattr(lib, f"volta_mi355x_fixed_{name}_device")
            assert fn(b.raw, None, *args) != 0 and fn(None, None, *args) != 0
        assert lib.volta_mi355x_fixed_weights_bytes(0, 1) == 0 and lib.volta_mi355x_fixed_weights_bytes(65536, 1) == 0
        assert lib.volta_mi355x_fixed_cache_bytes(1 << 31, 65535, 128, 65536) == 0  # over 2^64
        assert lib.volta_mi355x_fixed_cache_bytes(1 << 16, 64, 128, 65536) == (1 << 32) * (128 * 256 + 256)
        assert lib.volta_mi355x_fixed_cache_bytes(1 << 40, 1, 64, 64) == 0
