"""What the operators of generation refuse, on the host and before any device
work (no test here touches a device)."""

import ctypes

from tensorcrate_amd import lib
from tests.test_language_refusals import refused


def test_the_rotary_shape_is_the_headers():
    # Natural C alignment of `tc_rotary_shape`.
    assert lib.RotaryShape.epsilon.offset == 32 and lib.RotaryShape.tokens.offset == 40
    assert lib.RotaryShape.frequencies.offset == 56 and ctypes.sizeof(lib.RotaryShape) == 64 + 8 * 8


def test_rotary_norm():
    def shape(dtype=lib.F32, weight=lib.F32, tokens=10, heads=4, key_heads=2, size=16, count=16, pairs=lib.HALVES,
              normalize=True, epsilon=1e-5, positions=64, frequencies=64, query=(64, 16), key=(32, 16),
              query_out=(64, 16), key_out=(32, 16)):
        return lib.rotary(dtype, weight, tokens, heads, key_heads, size, count, pairs, normalize, epsilon, positions,
                          frequencies, query, key, query_out, key_out)

    forward = lambda given, *operands: refused("tc_rotary_norm", given, *(operands or [64] * 6))
    back = lambda given, *operands: refused("tc_rotary_norm_backward", given, *(operands or [64] * 10))
    for run, what in ((forward, "rotary norm"), (back, "rotary norm, backward")):
        assert run(None) == (lib.INVALID, f"{what}: no shape")
        assert run(shape(dtype=lib.F64)) == (lib.UNSUPPORTED, f"{what}: no kernel for f64")
        assert run(shape(dtype=lib.F16, weight=lib.BF16)) == (
            lib.UNSUPPORTED, f"{what}: no kernel for f16 heads with a bf16 weight")
        assert run(shape(size=0, count=0)) == (lib.INVALID, f"{what}: heads of no elements")
        assert run(shape(size=129, query=(516, 129), key=(258, 129), query_out=(516, 129), key_out=(258, 129))) == (
            lib.UNSUPPORTED, f"{what}: heads of 129 elements, more than 128")
        for count in (3, 18):
            assert run(shape(count=count)) == (lib.INVALID, f"{what}: {count} rotated of 16 elements")
        assert run(shape(pairs=2)) == (lib.INVALID, f"{what}: pairs of kind 2")
        for epsilon in (-1.0, float("nan"), float("inf")):
            assert run(shape(epsilon=epsilon))[0] == lib.INVALID
        assert run(shape(normalize=False)) == (lib.INVALID, f"{what}: a weight without a norm")
        for name in ("query", "key", "query_out", "key_out"):
            for steps in ((16, 16), (64, 15), (0, 16), (16, 0), (2**62, 16), (16, 2**62)):
                assert run(shape(**{name: steps}))[0] == lib.INVALID, (name, steps)
        assert run(shape(tokens=2**32))[0] == lib.UNSUPPORTED
        assert run(shape(frequencies=None)) == (lib.INVALID, f"{what}: a null operand")
    for missing in (0, 1, 4, 5):
        operands = [64] * 6
        operands[missing] = None
        assert forward(shape(), *operands) == (lib.INVALID, "rotary norm: a null operand")
    for missing in (0, 1, 2, 3, 6, 7):
        operands = [64] * 10
        operands[missing] = None
        assert back(shape(), *operands) == (lib.INVALID, "rotary norm, backward: a null operand")
    # Weights' gradients belong to the norm too.
    assert back(shape(normalize=False), 64, 64, None, None, None, None, 64, 64, 64, None)[0] == lib.INVALID
    # Nothing to do, and no device needed.
    assert forward(shape(tokens=0), *[None] * 6)[0] == lib.OK
    assert back(shape(tokens=0), *[None] * 10)[0] == lib.OK
