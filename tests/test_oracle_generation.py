"""The 64-bit gradients that the generation operators are tested against,
against differences of the 64-bit results."""

import numpy as np
import pytest

from tensorcrate_amd import lib
from tests import generation


@pytest.mark.parametrize("pairs", [lib.HALVES, lib.NEIGHBOURS])
@pytest.mark.parametrize("size,count,epsilon", [(8, 4, 0.1), (7, 2, 0.1), (6, 0, 0.1), (6, 3, None)])
def test_rotary_gradients_are_differences(size, count, epsilon, pairs):
    rng = np.random.default_rng(0)
    x, dz = (rng.standard_normal((3, 2, size)) for _ in range(2))
    weight = rng.standard_normal(size) if epsilon is not None else None
    positions, frequencies = np.array([0, 5, 900]), rng.uniform(0.01, 1.0, count)
    total = lambda: (generation.rotary(x, weight, epsilon, positions, frequencies, pairs)[0] * dz).sum()
    (dx, dw), _ = generation.rotary_backward(dz, x, weight, epsilon, positions, frequencies, pairs)
    step = 1e-5
    for values, gradient in ((x, dx), (weight, dw)):
        if values is None:
            continue
        for at in np.ndindex(values.shape):
            kept = values[at]
            values[at] = kept + step
            high = total()
            values[at] = kept - step
            low = total()
            values[at] = kept
            # The error of a central difference is of the order of step^2.
            assert abs((high - low) / (2 * step) - gradient[at]) < 1e-7 * (1 + abs(gradient[at]))


def test_a_turn_keeps_the_length_and_turns_back():
    rng = np.random.default_rng(1)
    y = rng.standard_normal((4, 2, 10))
    positions, frequencies = rng.integers(0, 2**32, 4), rng.uniform(0, 1, 4)
    for pairs in (lib.HALVES, lib.NEIGHBOURS):
        z, _ = generation.turned(y, positions, frequencies, pairs)
        assert np.allclose((z ** 2).sum(2), (y ** 2).sum(2), rtol=1e-13)
        assert np.allclose(generation.turned(z, positions, frequencies, pairs, back=True)[0], y, atol=1e-13)
        assert np.array_equal(z[..., 8:], y[..., 8:])
