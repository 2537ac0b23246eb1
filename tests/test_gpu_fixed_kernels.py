"""Every kernel of the fixed-point model operators at sizes that reach it: the
operators choose a kernel by sizes, and small cases take the same few.  Sizes
lie well inside the range of the kernel that they are for, on 256 CUs."""
import fixed_reference as ref
import numpy as np
import pytest
from test_gpu_fixed import (Held, attention_case, check_attention, exponentials, full, gen, normal, prompts,
                            run_attention, run_linear, want_attention)

pytestmark = pytest.mark.gpu

# rows, k, n for each shape of a product's tiles; 64 x 64 with four stages and
# with two, 128 x 128 with eight waves and with four
TILES = [(801, 131, 497), (1499, 99, 1201), (1543, 509, 1990), (4081, 199, 2033)]


def finished(acc, shift, *, bias=None, bias_shift=0, table=None, residual=None):
    """The epilogue over sums, in 64 bits."""
    if bias is not None:
        acc = acc + bias.astype(np.int64) * (1 << bias_shift)
    h = ref.sat(ref.rs(acc, shift))
    if table is not None:
        h = table.astype(np.int64)[h + 32768]
    if residual is not None:
        h = ref.sat(h + residual.astype(np.int64))
    return h.astype(np.int16)


class Product:
    """x w on the GPU with one upload for many calls."""

    def __init__(self, b, x, w, x_gap=0):
        self.b, self.rows, self.n = b, x.shape[0], w.shape[1]
        self.held = Held(b)
        wide = np.full((self.rows, x.shape[1] + x_gap), 12345, np.int16)
        wide[:, :x.shape[1]] = x
        self.x, self.stride = self.held.put(wide), x.shape[1] + x_gap
        self.packed = b.fixed_weights_device(self.held.put(w), *w.shape)
        self.held.keep(self.packed.storage)

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.held.__exit__()

    def __call__(self, shift=0, *, coarse=False, raw=False, out_gap=3, **kw):
        b = self.b
        with Held(b) as held:
            args = {k: held.put(v) if isinstance(v, np.ndarray) else v for k, v in kw.items()}
            stride = self.n + out_gap
            out = held.new(self.rows * stride, np.int64 if raw else np.int16, 31)
            if coarse:
                assert b.lib.volta_cuda_begin_coarse_timing(b.raw, 0) == 0
            b.fixed_linear_device(self.x, self.rows, self.packed, shift, x_stride=self.stride, out=out, out_stride=stride,
                                  raw=raw, **args)
            if coarse:
                assert b.lib.volta_cuda_end_coarse_timing(b.raw) == 0
            got = b.download_device(out).reshape(self.rows, stride)
            assert (got[:, self.n:] == 31).all()
            return got[:, :self.n]


@pytest.mark.parametrize("rows,k,n", TILES)
def test_tiles_with_shifts_up_to_the_largest(backend, rows, k, n):
    """Both ways of a tile's epilogue, in 32 bits (shifts to 45 with biases shifted by at most 29) and in 64, at
    their ends."""
    g = gen(rows)
    x, w, bias = full(g, (rows, k)), full(g, (k, n)), full(g, n)
    acc = ref._sums(x, w)
    with Product(backend, x, w) as product:
        for shift, bias_shift in ((0, 0), (1, 0), (15, 3), (16, 0), (17, 29), (31, 0), (32, 29), (45, 29), (45, 30),
                                  (46, 29), (46, 46), (62, 46)):
            want = finished(acc, shift, bias=bias, bias_shift=bias_shift)
            assert np.array_equal(product(shift, bias=bias, bias_shift=bias_shift), want), (shift, bias_shift)


@pytest.mark.parametrize("rows,k,n", TILES)
def test_tiles_with_each_optional_part(backend, rows, k, n):
    g = gen(rows + 1)
    x, w = normal(g, (rows, k), 1000), normal(g, (k, n), 2000)
    acc = ref._sums(x, w)
    parts = dict(bias=full(g, n), table=full(g, 65536), residual=full(g, (rows, n)))
    with Product(backend, x, w) as product:
        assert np.array_equal(product(raw=True), acc)
        for use in range(8):
            kw = {name: parts[name] for i, name in enumerate(parts) if use >> i & 1}
            if "bias" in kw:
                kw["bias_shift"] = 10
            assert np.array_equal(product(13, **kw), finished(acc, 13, **kw)), sorted(kw)
        raw = product(raw=True, bias=parts["bias"], bias_shift=46)
        assert np.array_equal(raw, acc + parts["bias"].astype(np.int64) * (1 << 46))


@pytest.mark.parametrize("rows,k,n", TILES)
@pytest.mark.parametrize("top", [32639, 32640, 32767])
def test_tiles_with_some_blocks_of_large_weights(backend, rows, k, n, top):
    """Blocks of 16 columns that need the offset beside blocks of the same tile that do not."""
    g = gen(rows + top)
    x, w = full(g, (rows, k)), normal(g, (k, n), 2000)
    for c in (0, 5, 37, 130, n // 2, n - 1):
        w[g.integers(0, k), c] = top
    bias = full(g, n)
    acc = ref._sums(x, w)
    with Product(backend, x, w) as product:
        assert np.array_equal(product(raw=True), acc)
        assert np.array_equal(product(14, bias=bias, bias_shift=9), finished(acc, 14, bias=bias, bias_shift=9))


@pytest.mark.parametrize("rows,k,n", TILES)
@pytest.mark.parametrize("gap", [0, 5])
def test_tiles_of_rows_copied_through_registers(rows, k, n, gap):
    """Rows that are not aligned, where no workspace may be allocated to align them."""
    from volta_mi355x import Backend
    g = gen(rows + gap)
    x, w = full(g, (rows, k)), full(g, (k, n))
    kw = dict(bias=full(g, n), bias_shift=9, table=full(g, 65536), residual=full(g, (rows, n)))
    acc = ref._sums(x, w)
    with Backend(timing_policy=1) as b, Product(b, x, w, x_gap=gap) as product:
        assert np.array_equal(product(20, coarse=True, **kw), finished(acc, 20, **kw))
        assert np.array_equal(product(raw=True, coarse=True), acc)


@pytest.mark.parametrize("rows,k,n", TILES)
def test_tiles_of_strided_aligned_rows(backend, rows, k, n):
    """Foreign values past k in the last piece of every row."""
    g = gen(rows + 7)
    gap = -k % 8 + 16
    x, w = full(g, (rows, k)), full(g, (k, n))
    acc = ref._sums(x, w)
    with Product(backend, x, w, x_gap=gap) as product:
        assert np.array_equal(product(raw=True), acc)
        assert np.array_equal(product(22), finished(acc, 22))


@pytest.mark.parametrize("rows,k,n", TILES)
def test_tiles_over_their_residual(backend, rows, k, n):
    g = gen(rows + 9)
    x, w, res = normal(g, (rows, k), 1000), normal(g, (k, n), 2000), full(g, (rows, n))
    want = finished(ref._sums(x, w), 13, residual=res)
    with Product(backend, x, w) as product, Held(backend) as held:
        dr = held.put(res)
        backend.fixed_linear_device(product.x, rows, product.packed, 13, residual=dr, out=dr)
        assert np.array_equal(backend.download_device(dr).reshape(rows, n), want)


@pytest.mark.parametrize("rows,n", [(801, 497), (1700, 1901)])
def test_tiles_with_the_longest_sums_of_equal_values(backend, rows, n):
    """k = 65,535 equal products, one column in each block of 16 apart: the i32 sums and the epilogue's 32-bit
    arithmetic at their ends."""
    k = 65535
    g = gen(rows)
    bias = full(g, n)
    for a, v in ((-32768, -32768), (-32768, 32767), (32767, 32767), (32767, 32639), (127, -129)):
        w = np.full((k, n), v, np.int16)
        w[:, ::16] = -32768
        column = np.where(np.arange(n) % 16 == 0, -32768, v).astype(np.int64)
        acc = np.broadcast_to(k * a * column, (rows, n))
        with Product(backend, np.full((rows, k), a, np.int16), w) as product:
            assert np.array_equal(product(raw=True), acc)
            for shift, bias_shift in ((16, 0), (32, 29), (45, 29)):
                want = finished(acc, shift, bias=bias, bias_shift=bias_shift)
                assert np.array_equal(product(shift, bias=bias, bias_shift=bias_shift), want), (a, v, shift)


# ---- attention: one team a workgroup takes over 512 workgroups of 128 rows -----------------------

@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [40, 64])
def test_attention_one_team(backend, dim, causal):
    g = gen(dim + causal)
    counts, lengths = prompts(g, 20, 300)
    check_attention(backend, dim, counts, lengths, 32, 32, dim, causal=causal)


@pytest.mark.parametrize("dim", [57, 64])
def test_attention_one_team_over_a_past_with_gaps(backend, dim):
    counts, lengths = prompts(gen(dim), 20, 260, past=150)
    check_attention(backend, dim, counts, lengths, 32, 32, dim, gap=9, q_offset=3)


@pytest.mark.parametrize("key", [32639, 32640])
def test_attention_one_team_grouped_with_few_large_values(backend, key):
    g = gen(key)
    counts, lengths = prompts(g, 20, 280, past=70)
    q, k, v, past = attention_case(3, counts, lengths, 64, 16, 64)
    for t in [q, k] + [p for p, _ in past if len(p)]:
        flat = t.reshape(-1)
        flat[g.integers(0, flat.size, max(1, flat.size // 4000))] = key
    got = run_attention(backend, q, k, v, lengths, counts, past, exponentials(), 16)
    assert np.array_equal(got, want_attention(q, k, v, lengths, counts, past, exponentials(), 16))


@pytest.mark.parametrize("length", [4096, 4097])
def test_attention_scores_at_the_limit_of_lds(backend, length):
    """Four rows a unit over 64 tiles are the most scores that a workgroup keeps; one token more goes to memory."""
    lengths = [length] * 4 + [4096, 4000, 3001, 64, 1]
    check_attention(backend, length, [1] * 9, lengths, 32, 8, 128)


# ---- norm: more rows than workgroups take at once -----------------------------------------------

@pytest.mark.parametrize("rows,cols", [(17001, 33), (17001, 600), (9001, 1300), (4500, 2500), (4500, 5000), (2200, 8300)])
def test_norm_of_many_rows(backend, rows, cols):
    g = gen(rows + cols)
    x, res, gain, bias = normal(g, (rows, cols), 3000), normal(g, (rows, cols), 5000), full(g, cols), full(g, cols)
    b = backend
    with Held(b) as held:
        kept, out = held.new(rows * (cols + 3), np.int16, 5), held.new(rows * (cols + 1), np.int16, 6)
        b.fixed_norm_device(held.put(x), rows, cols, held.put(gain), 3, cols, bias=held.put(bias), residual=held.put(res),
                            sum_out=kept, sum_stride=cols + 3, out=out, out_stride=cols + 1)
        y, h = (b.download_device(t).reshape(rows, -1) for t in (out, kept))
    assert (y[:, cols:] == 6).all() and (h[:, cols:] == 5).all()
    want, want_h = ref.norm(x, gain, 3, cols, bias=bias, residual=res)
    assert np.array_equal(y[:, :cols], want) and np.array_equal(h[:, :cols], want_h)
