"""Prompts and then tokens through rotation, cache and attention, against the
same in 64 bits with the roundings that the calls state: rotated queries and
keys to the type, keys and values to 8 bits, results to the type.

What is left is told by the root of the mean square of all errors.  The results'
own rounding adds half a step over the root of 3.  The rotation's 32 bits, some
24 roundings of 2^-24, take a value to the other side of a rounding now and
then: with a chance of 24 * 2^-24 over half a step, 2^-11.4 in bf16 and 2^-8.4 in
f16, by a step, so that a score, a sum of 40 products of size 1 / 6.3 each, moves
by 2^-7 * 2^-5.7 and 2^-10 * 2^-4.2 over the roots of 40 and 6.3, below 2^-13; in 8
bits with 2^-12 at most, by a step of 3 / 127, below 2^-11.  In f32 it is
their own size: scores of at most 10 and sums of 70 terms, some 100 roundings."""

import numpy as np
import pytest

from tensorcrate_amd import lib
from tests import generation, language
from tests.common import KIND_NAMES, KINDS
from tests.language import ROUNDING, stored
from tests.test_gpu_generation import HEADS, KEY_HEADS, SIZE, Model

pytestmark = pytest.mark.gpu

LENGTHS, DECODED = [70, 33, 50], 9


def held(fmt, x):
    """What the cache gives back of these rows."""
    if fmt == lib.CACHE_PLAIN:
        return x
    entries, scales = generation.quantised(x)
    return entries.astype(np.float64) * scales.astype(np.float64)[..., None]


def exact(model, frequencies):
    results = []
    for rows in model.projections:
        positions = np.arange(len(rows))
        q, k = (stored(generation.rotary(x, w, 1e-5, positions, frequencies, lib.HALVES)[0], model.kind)
                for x, w in zip((rows[:, :HEADS], rows[:, HEADS:HEADS + KEY_HEADS]), model.weights))
        k, v = held(model.fmt, k), held(model.fmt, rows[:, HEADS + KEY_HEADS:])
        results.append(language.attention(q, k, v, [0, len(rows)], model.scale)[0])
    return results


def root_mean_square(x):
    return (x ** 2).mean() ** 0.5


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("fmt", [lib.CACHE_PLAIN, lib.CACHE_INT8])
def test_prompts_then_tokens_to_their_roundings(kind, fmt):
    model = Model(kind, fmt, LENGTHS)
    at = [n - DECODED for n in LENGTHS]
    got = [model.step([0] * 3, at)]
    for count in (3, 1, 1, 1, 1, 1, 1):
        got.append(model.step(at, [p + count for p in at]))
        at = [p + count for p in at]
    want, unturned = exact(model, model.frequencies), exact(model, 0 * model.frequencies)
    loose = 2.0**-11 if fmt == lib.CACHE_INT8 else 2.0**-13 if kind != lib.F32 else 2.0**-17
    for name, mine, rows in (("prompts", got[:1], slice(-DECODED)), ("tokens", got[1:], slice(-DECODED, None))):
        result = np.concatenate([np.concatenate([step[s] for step in mine]) for s in range(3)])
        expected, other = (np.concatenate([t[s][rows] for s in range(3)]) for t in (want, unturned))
        size = root_mean_square(expected)
        with np.errstate(divide="ignore"):  # (a 0 is exact)
            half_step = ROUNDING[kind] * 2.0 ** np.floor(np.log2(np.abs(expected)))
        bound = 1.1 * root_mean_square(half_step) / 3 ** 0.5 + loose * size
        assert root_mean_square(result - expected) < bound, name
        # The bound tells what is not there at all, or not rotated.
        assert min(size, root_mean_square(other - expected)) > 20 * bound, name
