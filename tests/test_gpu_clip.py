"""The norm over many tensors, and clipping by it, against 64 bits.

Squares are exact in 64 bits and their sum is off by 2^-53 for each of fewer
than 2^30 terms, so the norm's error is its rounding to 32 bits; a clipped
element is off by the factor's rounding, the product's and the type's."""

import numpy as np
import pytest

from tensorcrate_amd import lib
from tests.common import KIND_NAMES, KINDS
from tests.language import EPSILON_32, ROUNDING, TINY, Rows, near, stored

pytestmark = pytest.mark.gpu


def arrays(kinds, pointers, lens):
    n = len(kinds)
    return (lib.u32 * max(n, 1))(*kinds), (lib.vp * max(n, 1))(*pointers), (lib.u64 * max(n, 1))(*lens)


def run(tensors, limit, in_place=False, shifts=None):
    """Tensors of (kind, values): (outputs, norm)."""
    shifts = shifts or [0] * len(tensors)
    sources = [Rows(v[None], k, shift=s) for (k, v), s in zip(tensors, shifts)]
    outs = sources if in_place else [Rows.empty(1, v.size, k, shift=(s * 5 + 1) % 8)
                                     for (k, v), s in zip(tensors, shifts)]
    kinds, pointers, lens = arrays([k for k, _ in tensors], [s.ptr for s in sources], [v.size for _, v in tensors])
    outputs = (lib.vp * max(len(tensors), 1))(*[o.ptr for o in outs])
    norm = lib.Buffer.of(np.full(1, 7.0, np.float32))
    lib.call("tc_global_norm", len(tensors), kinds, pointers, lens, norm.ptr)
    alone = float(norm.download(np.float32)[0])
    lib.call("tc_clip_global_norm", len(tensors), kinds, pointers, lens, limit, outputs, norm.ptr)
    got = float(norm.download(np.float32)[0])
    assert got == alone or (np.isnan(got) and np.isnan(alone))
    return [o.read()[0] for o in outs], got


def check(tensors, limit, got):
    outs, norm = got
    want = np.sqrt(sum(float(np.dot(v, v)) for _, v in tensors))
    with np.errstate(over="ignore"):
        reached = want if np.isfinite(np.float32(want)) else np.inf  # what 32 bits hold of it
    near(np.array([norm]), np.array([reached]), 1.01 * EPSILON_32 * want + 2.0**-149, "norm")
    limit = float(np.float32(limit))
    factor = limit / want if want > limit and reached < np.inf else 1.0
    for k, ((kind, values), out) in enumerate(zip(tensors, outs)):
        exact = values * factor
        loose = 0.0 if factor == 1.0 else (ROUNDING[kind] + 2.02 * EPSILON_32) * np.abs(exact) + TINY[kind]
        near(out, exact, loose, f"tensor {k}")


def tensors_of(sizes, kinds, seed, scale=1.0):
    rng = np.random.default_rng(seed)
    return [(kinds[n % len(kinds)], stored(rng.standard_normal(size) * scale, kinds[n % len(kinds)]))
            for n, size in enumerate(sizes)]


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("size", [1, 2, 3, 7, 8, 9, 17, 100, 4095, 8191, 8192, 16384, 16385, 100003, 3000001])
def test_one_tensor(kind, size):
    for shift, limit in ((0, 0.5), (1, 1e6), (3, 1.25), (7, 0.0)):
        tensors = tensors_of([size], [kind], seed=shift)
        check(tensors, limit, run(tensors, limit, shifts=[shift]))
        check(tensors, limit, run(tensors, limit, in_place=True, shifts=[shift]))


@pytest.mark.parametrize("count", [2, 95, 96, 97, 139, 140, 141, 281, 400])
def test_many_tensors_of_every_type(count):
    rng = np.random.default_rng(count)
    sizes = [int(s) for s in np.exp(rng.uniform(0, 10, count))]
    sizes[count // 2] = 0
    tensors = tensors_of(sizes, [lib.BF16, lib.F32, lib.F16, lib.F32], seed=count, scale=0.1)
    shifts = [int(s) for s in rng.integers(0, 9, count)]
    for limit in (2.0, 1e9):
        check(tensors, limit, run(tensors, limit, shifts=shifts))
    check(tensors, 2.0, run(tensors, 2.0, in_place=True, shifts=shifts))


def test_no_elements():
    assert run([], 1.0) == ([], 0.0)
    outs, norm = run([(lib.F32, np.zeros(0)), (lib.BF16, np.zeros(0))], 1.0)
    assert norm == 0.0 and all(o.size == 0 for o in outs)
    outs, norm = run([(lib.F32, np.zeros(40))], 0.0)
    assert norm == 0.0 and not outs[0].any()


def test_squares_past_and_below_32_bits():
    for scale in (1e25, 1e-30):
        tensors = [(lib.F32, stored(np.array([3.0, -4.0, 12.0]) * scale, lib.F32))]
        check(tensors, scale, run(tensors, scale))
    tensors = [(lib.BF16, stored(np.full(5000, 3e37), lib.BF16))]
    check(tensors, 1.0, run(tensors, 1.0))


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_a_norm_that_is_not_finite_scales_nothing(value):
    tensors = tensors_of([500, 20000], [lib.F32, lib.F16], seed=1)
    tensors[1][1][777] = value
    for in_place in (False, True):
        outs, norm = run(tensors, 1.0, in_place=in_place)
        assert not np.isfinite(norm)
        for (_, values), out in zip(tensors, outs):
            assert np.array_equal(values, out, equal_nan=True)


def test_the_same_bits_again():
    tensors = tensors_of([3000001, 77, 1000000], [lib.F32, lib.BF16, lib.F16], seed=3)
    (first, norm), (again, norm_again) = (run(tensors, 1.0) for _ in range(2))
    assert norm == norm_again and all(np.array_equal(a, b) for a, b in zip(first, again))


def test_the_norm_does_not_depend_on_where_a_tensor_starts():
    # 64 runs of one 2^-3 and seven 2^-30 behind it, whose squares vanish one
    # by one beside the first and together would be two units of the sum's last
    # place, and 2^-23 + 2^-48 more: all but those seven come to the square of
    # a number halfway between two of 32 bits, so that every unit of the sum's
    # last place shows in the norm's.
    values = np.full((64, 8), 2.0**-30)
    values[:, 0] = 2.0**-3
    values = np.concatenate([values.reshape(-1), [2.0**-12, 2.0**-12, 2.0**-24]])
    for kind in (lib.BF16, lib.F32):
        norms = {run([(kind, stored(values, kind))], 1e9, shifts=[shift])[1] for shift in range(9)}
        assert len(norms) == 1, (KIND_NAMES[kind], norms)
