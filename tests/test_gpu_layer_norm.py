"""Layer norm and its gradients against the plain forms in 64 bits.

Bounds: sums of n terms in f32, at most 16 in a row in a lane, 6 more over a
wave and 16 over a block (a long row's lane n/1024), are off by at most 40
(n/256) roundings of the sum of magnitudes, which 2^-17 (128 roundings) covers
for the rows here; then one rounding to the type.  A sum over rows is off by a
rounding for each row that one lane adds and each part that is added."""

import numpy as np
import pytest

from tensorcrate_amd import lib
from tests import language
from tests.common import KIND_NAMES, KINDS
from tests.language import EPSILON_32, ROUNDING, TINY, Rows, near, stored

pytestmark = pytest.mark.gpu

F32_SUMS = 2.0**-17
EPSILON = 1e-5

# Rows and columns: one element, one word more or less, the lanes of each
# form and one past them, many rows, long rows past a block's registers.
SHAPES = [(1, 1), (3, 2), (5, 7), (4, 8), (4, 9), (33, 31), (17, 64), (65, 65), (9, 127), (9, 128), (100, 129),
          (31, 257), (7, 511), (7, 513), (300, 1000), (40, 1027), (5, 2050), (3, 4096), (3, 4099), (2, 8192),
          (2, 8193), (2, 9300), (2, 12300), (2, 15000), (2, 16384), (2, 16391), (3, 40003), (5000, 24), (2500, 200)]


def inputs(kind, weight_kind, rows, cols, seed):
    rng = np.random.default_rng(seed)
    x = stored(rng.standard_normal((rows, cols)) * 2 + 0.5, kind)
    weight = stored(rng.uniform(0.5, 1.5, cols), weight_kind)
    bias = stored(rng.standard_normal(cols) * 0.1, weight_kind)
    dy = stored(rng.standard_normal((rows, cols)), kind)
    return x, weight, bias, dy


def forward(kind, weight_kind, x, weight, bias, gap=0, shift=0, in_place=False, statistics=True):
    rows, cols = x.shape
    source = Rows(x, kind, gap, shift)
    out = source if in_place else Rows.empty(rows, cols, kind, gap=(gap + 3) % 5, shift=(shift + 1) % 3)
    held = [None if v is None else Rows(v[None], weight_kind) for v in (weight, bias)]
    means, scales = (lib.Buffer(4 * rows) if statistics else None for _ in range(2))
    lib.call("tc_layer_norm", kind, weight_kind, source.ptr, source.step, rows, cols,
             *[None if h is None else h.ptr for h in held], EPSILON, out.ptr, out.step,
             *[None if b is None else b.ptr for b in (means, scales)])
    y = out.read()
    if not statistics:
        return y, None, None
    return y, means.download(np.float32), scales.download(np.float32)


def check_forward(kind, x, weight, bias, got):
    y, means, scales = got
    one, none = np.ones(x.shape[1]), np.zeros(x.shape[1])
    weight, bias = one if weight is None else weight, none if bias is None else bias
    want, mean, scale = language.layer_norm(x, weight, bias, EPSILON)
    most = np.abs(x).max(1)
    loose = F32_SUMS * most * scale  # of u: the mean's error, scaled
    # Scale's own error is the variance's: (mean's error)^2 vanishes beside it.
    bound = ROUNDING[kind] * np.abs(want) + TINY[kind] + (
        loose[:, None] * np.abs(weight) + F32_SUMS * (np.abs((want - bias)) + np.abs(bias)))
    near(y, want, bound, "y")
    if means is not None:
        near(means, mean, F32_SUMS * most, "means")
        near(scales, scale, (F32_SUMS + (loose * loose)) * scale, "scales")


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(kind, shape):
    for n, weight_kind in enumerate(sorted({kind, lib.F32})):
        x, weight, bias, _ = inputs(kind, weight_kind, *shape, seed=n)
        gap, shift = (0, 0) if n == 0 else (3, 1)
        check_forward(kind, x, weight, bias, forward(kind, weight_kind, x, weight, bias, gap, shift))


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("shape", [(5, 7), (9, 130), (6, 1029), (2, 17001)], ids=str)
def test_forward_in_place_and_without_operands(kind, shape):
    x, weight, bias, _ = inputs(kind, kind, *shape, seed=5)
    check_forward(kind, x, weight, bias, forward(kind, kind, x, weight, bias, gap=5, in_place=True))
    check_forward(kind, x, weight, None, forward(kind, kind, x, weight, None))
    check_forward(kind, x, None, bias, forward(kind, kind, x, None, bias, statistics=False))
    check_forward(kind, x, None, None, forward(kind, kind, x, None, None))


@pytest.mark.parametrize("cols", [5, 700, 20000])
def test_rows_of_one_value_and_of_none_finite(cols):
    x = np.full((4, cols), 3.25)
    x[1, cols // 2] = np.inf
    x[2, 0] = np.nan
    y, means, scales = forward(lib.F32, lib.F32, x, np.ones(cols), np.full(cols, 0.5))
    # A constant row has no deviation but the rounding of its mean.
    near(y[[0, 3]], np.full((2, cols), 0.5), F32_SUMS * 3.25 / np.sqrt(EPSILON), "constant rows")
    assert np.isnan(y[1]).any() and np.isnan(y[2]).all() and np.isinf(means[1]) and np.isnan(means[2])


def test_variance_of_rows_far_from_zero():
    # Deviations of 1 about 4096: a sum of squares would leave no bits of them.
    rng = np.random.default_rng(3)
    x = stored(4096 + rng.standard_normal((6, 3001)), lib.F32)
    check_forward(lib.F32, x, np.ones(3001), None, forward(lib.F32, lib.F32, x, np.ones(3001), None))
    _, _, scales = forward(lib.F32, lib.F32, x, None, None)
    near(scales, language.layer_norm(x, 1, 0, EPSILON)[2], 1e-5, "scales")


def backward(kind, weight_kind, dy, x, weight, mean, scale, gap=0, shift=0, in_place=False,
             wanted=("dx", "dweight", "dbias")):
    rows, cols = x.shape
    dy_rows, x_rows = Rows(dy, kind, gap, shift), Rows(x, kind, (gap + 2) % 7, shift)
    out = {"dx": dy_rows if in_place else Rows.empty(rows, cols, kind, gap=gap, shift=shift),
           "dweight": Rows.empty(1, cols, weight_kind, shift=shift), "dbias": Rows.empty(1, cols, weight_kind)}
    held = None if weight is None else Rows(weight[None], weight_kind)
    means, scales = (lib.Buffer.of(v.astype(np.float32)) for v in (mean, scale))
    ptr = lambda name: out[name].ptr if name in wanted else None
    lib.call("tc_layer_norm_backward", kind, weight_kind, dy_rows.ptr, dy_rows.step, x_rows.ptr, x_rows.step, rows,
             cols, None if held is None else held.ptr, means.ptr, scales.ptr, ptr("dx"), out["dx"].step,
             ptr("dweight"), ptr("dbias"))
    return {name: out[name].read() for name in wanted}


def check_backward(kind, weight_kind, dy, x, weight, got, mean, scale):
    weight = np.ones(x.shape[1]) if weight is None else weight
    mean, scale = (v.astype(np.float32).astype(np.float64) for v in (mean, scale))
    dx, dw, db = language.layer_norm_backward(dy, x, weight, mean, scale)
    u = np.abs(x - mean[:, None]) * scale[:, None]
    # u's own error: the difference of x and the mean, rounded once.
    du = 4 * EPSILON_32 * (u + (np.abs(x) + np.abs(mean)[:, None]) * scale[:, None])
    g = np.abs(dy * weight)
    if "dx" in got:
        loose = scale[:, None] * F32_SUMS * (g + g.mean(1, keepdims=True) + u * (g * u).mean(1, keepdims=True))
        loose += scale[:, None] * (du * (g * u).mean(1, keepdims=True) + u * (g * du).mean(1, keepdims=True))
        near(got["dx"], dx, ROUNDING[kind] * np.abs(dx) + TINY[kind] + loose, "dx")
    adds = (64 + x.shape[0] / 256 + 32) * EPSILON_32
    rounding = ROUNDING[weight_kind]
    if "dweight" in got:
        bound = rounding * np.abs(dw) + TINY[weight_kind] + adds * (np.abs(dy) * u).sum(0) + (np.abs(dy) * du).sum(0)
        near(got["dweight"][0], dw, bound, "dweight")
    if "dbias" in got:
        near(got["dbias"][0], db, rounding * np.abs(db) + TINY[weight_kind] + adds * np.abs(dy).sum(0), "dbias")


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_backward(kind, shape):
    for n, weight_kind in enumerate(sorted({kind, lib.F32})):
        x, weight, bias, dy = inputs(kind, weight_kind, *shape, seed=n + 10)
        _, mean, scale = language.layer_norm(x, weight, bias, EPSILON)
        gap, shift = (0, 0) if n == 0 else (3, 1)
        got = backward(kind, weight_kind, dy, x, weight, mean, scale, gap, shift)
        check_backward(kind, weight_kind, dy, x, weight, got, mean, scale)


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("shape", [(5, 7), (9, 130), (6, 1029), (2, 17001)], ids=str)
def test_backward_in_place_and_in_part(kind, shape):
    x, weight, bias, dy = inputs(kind, kind, *shape, seed=20)
    _, mean, scale = language.layer_norm(x, weight, bias, EPSILON)
    got = backward(kind, kind, dy, x, weight, mean, scale, gap=4, in_place=True)
    check_backward(kind, kind, dy, x, weight, got, mean, scale)
    for wanted in (("dx",), ("dweight",), ("dbias",), ("dweight", "dbias")):
        got = backward(kind, kind, dy, x, None, mean, scale, wanted=wanted)
        check_backward(kind, kind, dy, x, None, got, mean, scale)


def test_the_same_bits_again_and_zeros_for_no_rows():
    x, weight, bias, dy = inputs(lib.BF16, lib.F32, 3000, 777, seed=2)
    _, mean, scale = language.layer_norm(x, weight, bias, EPSILON)
    first, again = (backward(lib.BF16, lib.F32, dy, x, weight, mean, scale) for _ in range(2))
    for name, value in first.items():
        assert np.array_equal(value, again[name]), name
    out = Rows.empty(1, 9, lib.F32)
    lib.call("tc_layer_norm_backward", lib.F32, lib.F32, None, 9, None, 9, 0, 9, None, None, None, None, 9, out.ptr,
             None)
    assert np.array_equal(out.read(), np.zeros((1, 9)))
    lib.call("tc_layer_norm", lib.F32, lib.F32, None, 9, 0, 9, None, None, EPSILON, None, 9, None, None)
