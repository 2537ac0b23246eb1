"""Binary points of the fixed-point decoder's tensors, on the host."""
import pytest
from volta_mi355x import InvalidInput, forward

SIZES = dict(layers=2, heads=4, kv_heads=2, dim=16, hidden=32, vocab=50, positions=24)


def test_binary_points_of_the_tensors():
    """What is added to activations has their binary point; products, and the biases added to their sums, the weights'."""
    c = forward.FixedConfig(**SIZES, act_bits=9, weight_bits=12, gain_bits=11)
    want = {"wte": 12, "wpe": 9, "norm.gain": 11, "norm.bias": 9}
    for i in range(2):
        for name in ("qkv", "proj", "up", "down"):
            want[f"h{i}.{name}"] = want[f"h{i}.{name}.bias"] = 12
        for name in ("norm1", "norm2"):
            want[f"h{i}.{name}.gain"], want[f"h{i}.{name}.bias"] = 11, 9
    assert {name: c.bits(name) for name in c.shapes()} == want
    with pytest.raises(InvalidInput):
        c.bits("h2.qkv")


@pytest.mark.parametrize("act,weight,gain", [(-1, 13, 12), (16, 16, 16), (10, -1, 12), (10, 47, 12), (10, 13, 9), (2, 13, 18)])
def test_binary_points_that_the_operators_cannot_keep(act, weight, gain):
    with pytest.raises(InvalidInput):
        forward.FixedConfig(**SIZES, act_bits=act, weight_bits=weight, gain_bits=gain)


@pytest.mark.parametrize("act,weight,scale,shift", [(10, 13, 1, 3), (10, 10, 1, 0), (12, 9, 8, 0), (15, 0, 1 << 15, 0)])
def test_embeddings_come_to_the_activations_binary_point(act, weight, scale, shift):
    c = forward.FixedConfig(**SIZES, act_bits=act, weight_bits=weight, gain_bits=act)
    assert (c.embed_scale, c.embed_shift) == (scale, shift)
