"""Log probabilities, entropies, top tokens and the gradient of the logits
against the plain forms in 64 bits.

Bounds: a term's exponent (x - m) log2 e is off by two roundings of |x| log2 e
and of the largest |x| log2 e at most, and 2^v by 2 units; the sums of a row's
terms by one rounding for each that a lane adds (at most cols / 256 + 32) and
the joins'.  So the sum is off relatively by (8 max|x| + cols / 256 + 64) of
2^-24, which is what its logarithm, the normalizer, is off by absolutely beside
its own rounding; the mean of x - m in the entropy by that relatively, of at
most max - min."""

import numpy as np
import pytest

from tensorcrate_amd import lib
from tests import language
from tests.common import KIND_NAMES, KINDS
from tests.language import EPSILON_32, ROUNDING, TINY, Rows, near, stored

pytestmark = pytest.mark.gpu

NONE = 0xFFFFFFFF
# Rows and columns: one logit, a word more or less, one batch of a block
# (8192 or 4096) and one past it, long rows split over blocks, many rows.
SHAPES = [(1, 1), (3, 2), (2, 7), (5, 8), (4, 9), (3, 63), (7, 100), (2, 255), (3, 257), (2, 1024), (2, 4095), (2, 4097),
          (2, 8192), (3, 8193), (1, 33000), (16, 50001), (3, 131072), (1100, 1000), (1030, 9001), (4000, 17)]


def inputs(kind, rows, cols, seed, spread=3.0, masked=0):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, cols)) * spread
    tokens = rng.integers(0, cols, rows).astype(np.uint32)
    x[np.arange(rows), tokens] += rng.uniform(0, 12, rows)
    if masked:
        x[:, cols - masked:] = -np.inf
    tokens[rng.random(rows) < 0.2] = NONE
    return stored(x, kind), tokens


def run(kind, x, tokens, top, gap=0, shift=0, parts=("given", "normalizers", "entropies")):
    rows, cols = x.shape
    logits = Rows(x, kind, gap, shift, around=np.inf)
    held = lib.Buffer.of(tokens.astype(np.uint32))
    out = {name: lib.Buffer(4 * rows) for name in ("given", "normalizers", "entropies")}
    top_p, top_t = lib.Buffer(4 * rows * max(top, 1)), lib.Buffer(4 * rows * max(top, 1))
    ptr = lambda name: out[name].ptr if name in parts else None
    lib.call("tc_log_probabilities", kind, logits.ptr, logits.step, rows, cols, held.ptr if "given" in parts else None,
             ptr("given"), ptr("normalizers"), ptr("entropies"), top, top_p.ptr if top else None,
             top_t.ptr if top else None)
    got = {name: out[name].download(np.float32).astype(np.float64) for name in parts}
    if top:
        got["top"] = top_p.download(np.float32, rows * top).reshape(rows, top).astype(np.float64)
        got["tokens"] = top_t.download(np.uint32, rows * top).reshape(rows, top)
    return got


def check(x, tokens, top, got):
    cols = x.shape[1]
    given, normalizers, entropies, top_p, top_t = language.log_probabilities(x, tokens, top)
    finite = np.where(np.isfinite(x), x, 0.0)
    large, spread = np.abs(finite).max(1), finite.max(1) - finite.min(1)
    sums = (8 * large + cols / 256 + 64) * EPSILON_32
    if "normalizers" in got:
        near(got["normalizers"], normalizers, sums + 2 * EPSILON_32 * np.abs(normalizers), "normalizers")
    if "given" in got:
        near(got["given"], given, sums + 4 * EPSILON_32 * (spread + large), "log probabilities")
    if "entropies" in got:
        near(got["entropies"], entropies, 2 * sums * (1 + np.log(cols) + np.minimum(spread, 50)), "entropies")
    if top:
        near(got["top"], top_p, (sums + 4 * EPSILON_32 * (spread + large))[:, None], "top log probabilities")
        assert np.array_equal(got["tokens"], top_t)


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(kind, shape):
    rows, cols = shape
    x, tokens = inputs(kind, rows, cols, seed=1, masked=cols // 5)
    check(x, tokens, 0, run(kind, x, tokens, 0))
    for top in sorted({1, min(5, cols), min(64, cols)}):
        check(x, tokens, top, run(kind, x, tokens, top, gap=(3 * top) % 7, shift=top % 3))


@pytest.mark.parametrize("cols", [70, 8192, 30000, 131073])
@pytest.mark.parametrize("rows", [1, 1100])
@pytest.mark.parametrize("shape", ["rising", "falling", "equal", "two values", "steps", "signed zeros"])
def test_top_of_rows_in_order(shape, rows, cols):
    if rows * cols > 40_000_000:
        rows = 300
    at = np.arange(cols)
    row = {"rising": at * 2.0**-12, "falling": -at * 2.0**-12, "equal": np.full(cols, 1.5),
           "two values": np.where(at % 1000 == 999, 2.0, 1.0), "steps": (at // 64) * 2.0**-8,
           "signed zeros": np.where(at % 2 == 0, -0.0, 0.0)}[shape]
    x = stored(np.repeat(row[None], rows, 0), lib.F32)
    tokens = np.zeros(rows, np.uint32)
    for top in (7, 64):
        check(x, tokens, top, run(lib.F32, x, tokens, top))


@pytest.mark.parametrize("cols", [40, 9000, 60000])
def test_rows_with_nothing_or_no_number(cols):
    x, tokens = inputs(lib.F32, 6, cols, seed=4)
    tokens[:] = 3
    x[0] = -np.inf
    x[1, cols - 1] = np.nan
    x[2, 3:] = np.nan
    x[3, 5] = np.inf
    x[4] = -np.inf
    x[4, 17] = 2.0
    got = run(lib.F32, x, tokens, 20)
    given, normalizers, entropies, top_p, top_t = language.log_probabilities(x, tokens, 20)
    assert np.array_equal(got["tokens"], top_t)
    assert np.isneginf(got["given"][[0, 4]]).all() and got["entropies"][0] == 0 and np.isneginf(got["normalizers"][0])
    assert np.isneginf(got["top"][0]).all()
    assert np.isnan(got["normalizers"][[1, 2, 3]]).all() and np.isnan(got["given"][[1, 2]]).all()
    near(got["normalizers"][4:], normalizers[4:], 1e-5, "normalizers")
    near(got["entropies"][4:], entropies[4:], 1e-5, "entropies")
    assert got["top"][4, 0] == 0 and np.isneginf(got["top"][4, 1:]).all()


def test_results_left_out():
    x, tokens = inputs(lib.BF16, 5, 3000, seed=6)
    for parts in (("given",), ("normalizers",), ("entropies",), ()):
        for top in (0, 3):
            check(x, tokens, top, run(lib.BF16, x, tokens, top, parts=parts))


def test_large_logits():
    # Far from zero, as a constant added to every logit: nothing overflows.
    x, tokens = inputs(lib.F32, 3, 5000, seed=8)
    far = stored(x + 3e4, lib.F32)
    check(far, tokens, 5, run(lib.F32, far, tokens, 5))
    far = stored(x * 1e30, lib.F32)
    got = run(lib.F32, far, tokens, 5)
    assert np.array_equal(got["tokens"], language.log_probabilities(far, tokens, 5)[4])
    assert np.isfinite(got["normalizers"]).all()


def backward(kind, x, tokens, normalizers, entropies, d_given, d_entropies, gap=0, shift=0, in_place=False):
    rows, cols = x.shape
    logits = Rows(x, kind, gap, shift, around=7.0)
    out = logits if in_place else Rows.empty(rows, cols, kind, (gap + 2) % 5, (shift + 1) % 3)
    held = [lib.Buffer.of(tokens.astype(np.uint32))] + [
        None if v is None else lib.Buffer.of(v.astype(np.float32)) for v in (normalizers, entropies, d_given, d_entropies)]
    lib.call("tc_log_probabilities_backward", kind, logits.ptr, logits.step, rows, cols,
             *[None if h is None else h.ptr for h in held], out.ptr, out.step)
    return out.read()


def check_backward(kind, x, tokens, normalizers, entropies, d_given, d_entropies, got):
    zeros = np.zeros(x.shape[0])
    g, h = (zeros if d is None else d for d in (d_given, d_entropies))
    entropies = zeros if entropies is None else entropies
    want = language.log_probabilities_backward(x, tokens, normalizers, entropies, g, h)
    with np.errstate(invalid="ignore"):
        log_p = np.where(np.isneginf(normalizers)[:, None], -np.inf, x - normalizers[:, None])
    p = np.exp(log_p)
    finite = np.where(p == 0, 0.0, log_p)
    size = p * (np.abs(g)[:, None] + np.abs(h)[:, None] * (np.abs(finite) + np.abs(entropies)[:, None]))
    # The exponent is off by two roundings of itself and one of its parts.
    exponent = 4 * EPSILON_32 * (np.abs(finite) + 2)
    loose = size * (exponent + 8 * EPSILON_32) + 2 * EPSILON_32 * np.abs(want)
    near(got, want, ROUNDING[kind] * np.abs(want) + 2 * TINY[kind] + loose + 1e-37, "d logits")


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_backward(kind, shape):
    rows, cols = shape
    rng = np.random.default_rng(3)
    x, tokens = inputs(kind, rows, cols, seed=2, masked=cols // 5)
    _, normalizers, entropies, _, _ = language.log_probabilities(x, tokens, 0)
    normalizers, entropies, g, h = (v.astype(np.float32).astype(np.float64) for v in (
        normalizers, entropies, rng.standard_normal(rows), rng.standard_normal(rows)))
    g[rng.random(rows) < 0.1] = 0
    for given, spread, n in ((g, None, 0), (None, h, 1), (g, h, 2)):
        got = backward(kind, x, tokens, normalizers, None if spread is None else entropies, given, spread, gap=n,
                       shift=n, in_place=n == 2)
        check_backward(kind, x, tokens, normalizers, None if spread is None else entropies, given, spread, got)


def test_backward_of_rows_with_nothing():
    x, tokens = inputs(lib.F32, 4, 500, seed=9)
    tokens[:] = [1, 2, NONE, 3]
    x[0] = -np.inf
    x[2, 7] = np.nan
    _, normalizers, _, _, _ = language.log_probabilities(x, tokens, 0)
    normalizers[2] = np.nan
    got = backward(lib.F32, x, tokens, normalizers, None, np.ones(4), None)
    assert np.array_equal(got[[0, 2]], np.zeros((2, 500)))
    check_backward(lib.F32, x[[1, 3]], tokens[[1, 3]], normalizers[[1, 3]].astype(np.float32).astype(np.float64), None,
                   np.ones(2), None, got[[1, 3]])


def test_no_rows():
    lib.call("tc_log_probabilities", lib.F32, None, 9, 0, 9, None, None, None, None, 0, None, None)
    lib.call("tc_log_probabilities_backward", lib.F32, None, 9, 0, 9, None, None, None, None, None, None, 9)


# The lowest finite numbers of the types, and others that masks are made with.
FINITE_MASKS = [(lib.F32, -np.finfo(np.float32).max), (lib.F32, -1e38), (lib.F32, -1e37), (lib.F32, -1e9),
                (lib.F16, -65504.0), (lib.BF16, -3.3895313892515355e38), (lib.BF16, -1e38)]


@pytest.mark.parametrize("shape", [(3, 40), (3, 1000), (1, 33000), (2, 131072), (1100, 2050)], ids=str)
@pytest.mark.parametrize("kind, mask", FINITE_MASKS)
def test_logits_masked_with_a_number(kind, mask, shape):
    # Their probability is 0 in 64 bits and in 32, as that of -infinity is.
    rows, cols = shape
    column = np.arange(cols)
    x, tokens = inputs(kind, rows, cols, seed=11)
    for masked in (column >= cols - 40 // 2, column < cols // 2, column // 8 % 2 == 0, column != cols // 3):
        here = np.where(masked, stored(mask, kind), x)
        removed = np.where(masked, -np.inf, x)
        kept = np.flatnonzero(~masked).astype(np.uint32)
        given = np.where(tokens == NONE, NONE, kept[tokens.astype(np.int64) % len(kept)]).astype(np.uint32)
        top = min(5, len(kept))
        check(removed, given, 0, run(kind, here, given, 0))
        check(removed, given, top, run(kind, here, given, top))


@pytest.mark.parametrize("kind, mask", FINITE_MASKS)
@pytest.mark.parametrize("cols", [40, 33000])
def test_rows_of_nothing_but_a_masks_number(kind, mask, cols):
    # All alike, whatever the number: every token has the probability 1 / cols.
    x = stored(np.full((2, cols), mask), kind)
    got = run(kind, x, np.zeros(2, np.uint32), 3)
    sums = (cols / 256 + 64) * EPSILON_32
    near(got["entropies"], np.full(2, np.log(cols)), 2 * sums * (1 + np.log(cols)), "entropies")
    near(got["given"], np.full(2, -np.log(cols)), sums + 4 * EPSILON_32 * np.log(cols), "log probabilities")
    assert np.array_equal(got["tokens"], [[0, 1, 2]] * 2)


@pytest.mark.parametrize("kind, mask", [*FINITE_MASKS, (lib.F32, -np.inf), (lib.BF16, -np.inf)])
@pytest.mark.parametrize("slope", [1.0, 1e9])
def test_backward_of_masked_logits(kind, mask, slope):
    # An impossible token's gradient is 0, however large the entropy's is.
    if kind == lib.F16 and slope > 1:
        pytest.skip("the results themselves are past f16")
    rows, cols = 3, 9001
    x, tokens = inputs(kind, rows, cols, seed=12)
    masked = np.arange(cols) % 9 < 3
    here, removed = np.where(masked, stored(mask, kind), x), np.where(masked, -np.inf, x)
    tokens[:] = [3, NONE, 8]
    got = run(kind, here, tokens, 0)
    _, normalizers, entropies, _, _ = language.log_probabilities(removed, tokens, 0)
    normalizers, entropies = (v.astype(np.float32).astype(np.float64) for v in (normalizers, entropies))
    h = np.array([-slope, slope, slope])
    have = backward(kind, here, tokens, normalizers, entropies, np.ones(rows), h)
    check_backward(kind, removed, tokens, normalizers, entropies, np.ones(rows), h, have)
    assert not have[:, masked].any()
    assert np.isfinite(backward(kind, here, tokens, got["normalizers"], got["entropies"], np.ones(rows), h)).all()
