"""What the serving operators refuse before anything reaches the library: a backend without a GPU, whose library fails
the test when it is called."""
import ctypes

import numpy as np
import pytest
from volta_mi355x import FIXED_CHOICE, InvalidInput
from volta_mi355x.accel import Backend, DeviceBuffer, FixedKvCache


class NoLibrary:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


@pytest.fixture
def backend():
    b = Backend.__new__(Backend)
    b.raw, b.lib, b._live = ctypes.c_void_p(), NoLibrary(), {}

    def alloc(n, dtype):
        buf = DeviceBuffer(len(b._live) + 1, n, np.dtype(dtype), id(b))
        b._live[buf.id] = buf
        return buf

    b.alloc_device = alloc
    return b


def test_attention_windows_and_prefixes(backend):
    b = backend
    x, table = b.alloc_device(4096, np.int16), b.alloc_device(100, np.uint16)
    cache = FixedKvCache(b.alloc_device(1 << 20, np.uint8), 3, 2, 16, 70)
    seqs = [[0, 0, 1, 1]]
    for kw in (dict(window=-1), dict(window=3, sinks=-1), dict(sinks=2), dict(window=4, causal=False),
               dict(window=4, prefix=(1, 3)), dict(prefix=(3, 1)), dict(prefix=(-1, 1)), dict(prefix=(1, 71)),
               dict(prefix=(1, -1))):
        with pytest.raises(InvalidInput):
            b.fixed_attention_device(x, cache, seqs, 2, table, 12, **kw)


def test_rotations(backend):
    b = backend
    x, g, i = b.alloc_device(4096, np.int16), b.alloc_device(200, np.int16), b.alloc_device(64, np.int32)
    turn = dict(angles=x, angle_rows=4, positions=i)
    for args, kw in (((0, 2, 16), {}), ((4, 0, 16), {}), ((4, -1, 16), dict(kv_heads=2)), ((4, 2, 16), dict(kv_heads=-1)),
                     ((4, 2, 0), {}), ((4, 2, 129), {}), ((4, 65536, 1), {}), ((4, 2, 16), dict(gain_shift=16)),
                     ((4, 2, 16), dict(gain_shift=-1)), ((4, 2, 16), dict(angle_shift=16)), ((4, 2, 16), dict(eps=0)),
                     ((4, 2, 16), dict(eps=(1 << 40) + 1)), ((4, 2, 16), dict(turn, rotated=3)),
                     ((4, 2, 16), dict(turn, rotated=18)), ((4, 2, 16), dict(turn, rotated=-2)),
                     ((4, 2, 16), dict(turn, rotated=0)), ((4, 2, 16), dict(rotated=4)),
                     ((4, 2, 16), dict(turn, angle_rows=0)), ((4, 2, 16), dict(turn, positions=None)),
                     ((4, 2, 15), turn), ((4, 2, 16), dict(turn, angle_rows=257)), ((65, 2, 16), turn),
                     ((4, 2, 16), dict(turn, positions=x)), ((4, 2, 16), dict(turn, angles=i)),
                     ((4, 2, 16), dict(q_gain=i)), ((4, 2, 16), dict(k_gain=g, k_gain_offset=190)),
                     ((4, 2, 16), dict(x_stride=31)), ((4, 2, 16), dict(x_offset=4000)), ((200, 2, 16), {}),
                     ((4, 2, 16), dict(out=i)), ((4, 2, 16), dict(out=x, out_stride=20)), ((4, 2, 16), dict(out_offset=1))):
        with pytest.raises(InvalidInput):
            b.fixed_rotate_device(x, *args, **kw)


def choices(n, **kw):
    c = np.zeros(n, FIXED_CHOICE)
    c["mask"], c["repetition"] = -1, 65536
    for name, value in kw.items():
        c[name] = value
    return c


def test_choices(backend):
    b = backend
    l, i = b.alloc_device(4000, np.int64), b.alloc_device(100, np.int32)
    words = b.alloc_device(100, np.uint32)
    for args, kw in (((0, 10), {}), ((2, 0), {}), ((1, (1 << 24) + 1), {}), ((41, 100), {}), ((2, 10), dict(logits_stride=9)),
                     ((2, 10), dict(bias_shift=47)), ((2, 10), dict(bias_shift=-1)), ((2, 10), dict(out=l)),
                     ((2, 10), dict(out=i, out_offset=99)), ((2, 10), dict(adjusted=i)),
                     ((2, 10), dict(adjusted=l, adjusted_offset=3990)), ((2, 10), dict(bias_tokens=i)),
                     ((2, 10, choices(3)), {}), ((2, 10, np.zeros((2, 8), np.int64)), {}), ((2, 10, [1, 2]), {}),
                     ((2, 10, choices(2, repetition=[1, 0])), {}), ((2, 10, choices(2, history_count=1)), {}),
                     ((2, 10, choices(2, history_count=101)), dict(history=i)),
                     ((2, 10, choices(2, history_first=100, history_count=1)), dict(history=i)),
                     ((2, 10, choices(2, history_first=(1 << 64) - 1, history_count=2)), dict(history=i)),
                     ((2, 10, choices(2, history_count=(1 << 24) + 1)), dict(history=i)),
                     ((2, 10, choices(2, history_count=4)), dict(history=l)),
                     ((2, 10, choices(2, history_count=4)), dict(history=i, history_offset=97)),
                     ((2, 10, choices(2, bias_count=1)), {}),
                     ((2, 10, choices(2, bias_count=101)), dict(bias_tokens=i, bias_values=i)),
                     ((2, 10, choices(2, bias_count=4)), dict(bias_tokens=i, bias_values=words)),
                     ((2, 10, choices(2, mask=0)), {}), ((2, 10, choices(2, mask=100)), dict(allowed=words)),
                     ((2, 33, choices(2, mask=50)), dict(allowed=words)), ((2, 10, choices(2, mask=0)), dict(allowed=l)),
                     ((2, 33, choices(2, mask=0)), dict(allowed=words, allowed_stride=1))):
        with pytest.raises(InvalidInput):
            b.fixed_choose_device(l, *args, **kw)


def test_unused_lists_may_start_anywhere(backend):
    """What reaches the library: rows without entries do not count, wherever their lists start."""
    b, calls = backend, []

    class Library:
        def volta_mi355x_fixed_choose_device(self, raw, args, choices, rows):
            calls.append((args.history_id, args.bias_tokens_id, rows))
            return 0

    b.lib = Library()
    l, i, out = b.alloc_device(400, np.int64), b.alloc_device(100, np.int32), b.alloc_device(9, np.int32)
    for n in (1, 2, 9):
        c = choices(n, history_first=(1 << 64) - 1, bias_first=1 << 63)
        b.fixed_choose_device(l, n, 10, c, out=out)
        c["history_first"][-1], c["history_count"][-1] = 98, 2
        b.fixed_choose_device(l, n, 10, c, history=i, out=out)
        c["bias_first"][-1], c["bias_count"][-1] = 0, 100
        b.fixed_choose_device(l, n, 10, c, history=i, bias_tokens=i, bias_values=i, out=out)
        c["history_first"][-1] = 99
        with pytest.raises(InvalidInput):
            b.fixed_choose_device(l, n, 10, c, history=i, bias_tokens=i, bias_values=i, out=out)
    assert calls == [(h * i.id, t * i.id, n) for n in (1, 2, 9) for h, t in ((0, 0), (1, 0), (1, 1))]


def test_entry_points_without_a_context_or_arguments():
    from volta_mi355x import load_library
    lib = load_library()
    assert lib.volta_mi355x_fixed_window_attention_device(None, None, None, 1, 0, None, 0) != 0
    assert lib.volta_mi355x_fixed_prefix_attention_device(None, None, None, 0, 1, None, 0) != 0
    assert lib.volta_mi355x_fixed_rotate_device(None, None) != 0
    assert lib.volta_mi355x_fixed_choose_device(None, None, None, 1) != 0


def test_fields_and_binary_points_of_a_served_model():
    from volta_mi355x import forward
    base = dict(layers=1, heads=4, kv_heads=2, dim=16, hidden=32, vocab=50, positions=24)
    for kw in (dict(rotary=3), dict(rotary=18), dict(rotary=-2), dict(rotary=4, rotary_base=0.0), dict(window=-1),
               dict(window=5, sinks=-1), dict(sinks=2)):
        with pytest.raises(InvalidInput):
            forward.FixedConfig(**base, **kw)
    c = forward.FixedConfig(**base, rotary=8, head_norm=True)
    assert set(forward.FixedConfig(**base).shapes()) - set(c.shapes()) == {"wpe"}
    assert {n: (s, c.bits(n)) for n, s in c.shapes().items() if n not in forward.FixedConfig(**base).shapes()} == {
        "h0.q_norm.gain": ((16,), 12), "h0.k_norm.gain": ((16,), 12)}
    # half a step of 2^-14 from the angles themselves
    table = forward.rotation_table(c) / 2.0 ** 14
    angles = np.arange(24)[:, None] * 10000.0 ** (-np.arange(4) / 4)
    assert table.shape == (24, 4, 2)
    assert np.abs(table - np.stack([np.cos(angles), np.sin(angles)], -1)).max() <= 2.0 ** -15
