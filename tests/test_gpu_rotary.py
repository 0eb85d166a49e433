"""The norm of heads with their rotation by position, and the gradients, against
the formulas in 64 bits."""

import itertools

import numpy as np
import pytest

from tensorcrate_amd import lib
from tests import generation
from tests.generation import Heads
from tests.language import EPSILON_32, ROUNDING, TINY, near, stored

pytestmark = pytest.mark.gpu

EPSILON = 1e-5
KINDS = [lib.F32, lib.F16, lib.BF16]


class Case:
    def __init__(self, kind, tokens, heads, key_heads, size, count, pairs, normalize=True, weight=None, positions=None,
                 layout={}, out_layout={}, weights=True, seed=0, frequencies=None):
        rng = np.random.default_rng(seed)
        self.kind, self.weight_kind, self.pairs = kind, kind if weight is None else weight, pairs
        self.normalize, self.epsilon = normalize, EPSILON if normalize else None
        self.positions = rng.integers(0, 5000, tokens).astype(np.uint32) if positions is None else np.asarray(
            positions, np.uint32)
        self.frequencies = (10000.0 ** (-np.arange(count // 2) / max(count // 2, 1))).astype(
            np.float32) if frequencies is None else frequencies
        self.shapes = [(tokens, heads, size), (tokens, key_heads, size)]
        self.x = [stored(rng.standard_normal(s) * 1.5, kind) for s in self.shapes]
        self.dz = [stored(rng.standard_normal(s) * 0.1, kind) for s in self.shapes]
        self.weights = [stored(rng.standard_normal(size) * 0.3 + 1, self.weight_kind)
                        if normalize and weights else np.ones(size) for _ in range(2)]
        self.held = [Heads(x, kind, **layout) for x in self.x]
        self.held_dz = [Heads(d, kind, **out_layout) for d in self.dz]
        self.out = [Heads.empty(*s, kind, **out_layout) for s in self.shapes]
        self.dx = [Heads.empty(*s, kind, **layout) for s in self.shapes]
        self.held_weights = [Heads(w.reshape(1, 1, size), self.weight_kind, shift=1) for w in self.weights]
        self.dw = [Heads.empty(1, 1, size, self.weight_kind, shift=3) for _ in range(2)]
        self.device = [lib.Buffer.of(self.positions), lib.Buffer.of(self.frequencies)]
        self.given = [h.ptr if normalize and weights else None for h in self.held_weights]
        self.shape = lib.rotary(kind, self.weight_kind, tokens, heads, key_heads, size, count, pairs, normalize,
                                EPSILON, self.device[0].ptr, self.device[1].ptr if count else None,
                                self.held[0].steps, self.held[1].steps, self.out[0].steps, self.out[1].steps)

    def far(self):
        """By how much an angle of 64 bits may be off: three roundings."""
        most = float(self.positions.max(initial=0)) * float(np.abs(self.frequencies).max(initial=0.0))
        return most * 2.0 ** -51

    def forward(self):
        lib.call("tc_rotary_norm", self.shape, *(h.ptr for h in self.held), *self.given, *(o.ptr for o in self.out))

    def backward(self, dw=True):
        sums = [d.ptr if dw and self.normalize else None for d in self.dw]
        lib.call("tc_rotary_norm_backward", self.shape, *(d.ptr for d in self.held_dz), *(h.ptr for h in self.held),
                 *self.given, *(d.ptr for d in self.dx), *sums)

    def check_forward(self, got=None):
        for n in range(2):
            z, sizes = generation.rotary(self.x[n], self.weights[n], self.epsilon, self.positions, self.frequencies,
                                         self.pairs)
            # In roundings of 32 bits: 12 of the mean of squares, halved by the
            # root, 4 of the root, the quotient and two products; 2 of the
            # angle's part of a turn (2 pi / 2^26), 4 of the functions, 2 here.
            bound = (24 * EPSILON_32 + self.far()) * sizes + ROUNDING[self.kind] * np.abs(z) + TINY[self.kind]
            near(self.out[n].read() if got is None else got[n].read(), z, bound, f"rotated {'queries keys'.split()[n]}")

    def check_backward(self, dw=True, got=None):
        for n in range(2):
            (dx, weight), (sizes, weight_sizes) = generation.rotary_backward(
                self.dz[n], self.x[n], self.weights[n], self.epsilon, self.positions, self.frequencies, self.pairs)
            # As forward, and 12 roundings more of the mean of g u.
            bound = (40 * EPSILON_32 + 2 * self.far()) * sizes + ROUNDING[self.kind] * np.abs(dx) + TINY[self.kind]
            near(self.dx[n].read() if got is None else got[n].read(), dx, bound, f"gradient {n}")
            if self.normalize and dw:
                rows = self.shapes[n][0] * self.shapes[n][1]
                bound = ((24 + rows) * EPSILON_32 + self.far()) * weight_sizes + ROUNDING[self.weight_kind] * np.abs(
                    weight) + TINY[self.weight_kind]
                near(self.dw[n].read()[0, 0], weight, bound, f"weight's gradient {n}")


SIZES = [(128, 128), (128, 64), (80, 80), (80, 40), (64, 64), (96, 24), (20, 20), (37, 10), (36, 36), (6, 2), (1, 0),
         (2, 2), (127, 126), (75, 0), (128, 8)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pairs", [lib.HALVES, lib.NEIGHBOURS])
@pytest.mark.parametrize("size,count", SIZES)
def test_sizes(kind, pairs, size, count):
    for normalize in (True, False):
        case = Case(kind, 5, 3, 2, size, count, pairs, normalize)
        case.forward()
        case.check_forward()
        case.backward()
        case.check_backward()


LAYOUTS = [dict(gap=3, token_gap=5, shift=1), dict(gap=0, token_gap=0, turned=True), dict(gap=1, token_gap=7, shift=2,
                                                                                         turned=True)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("layout,out_layout", itertools.product(LAYOUTS, LAYOUTS[:2]))
def test_layouts(kind, layout, out_layout):
    case = Case(kind, 7, 4, 1, 48, 32, lib.HALVES, layout=layout, out_layout=out_layout, weight=lib.F32)
    case.forward()
    case.check_forward()
    case.backward()
    case.check_backward()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tokens,heads,key_heads", [(1, 1, 1), (1, 40, 8), (17, 0, 3), (17, 3, 0), (3000, 2, 1),
                                                    (9001, 1, 1), (300, 7, 7)])
def test_counts(kind, tokens, heads, key_heads):
    case = Case(kind, tokens, heads, key_heads, 24, 24, lib.NEIGHBOURS, weight=lib.F32)
    case.forward()
    case.check_forward()
    case.backward()
    case.check_backward()


def test_nothing():
    case = Case(lib.F32, 0, 2, 1, 16, 16, lib.HALVES)
    case.forward()
    case.backward()
    assert all((d.read() == 0).all() for d in case.dw)
    case = Case(lib.F32, 4, 0, 0, 16, 16, lib.HALVES)
    case.forward()
    case.backward()
    assert all((d.read() == 0).all() for d in case.dw)


@pytest.mark.parametrize("kind", KINDS)
def test_far_positions(kind):
    positions = [0, 1, 2**20, 2**24 + 1, 2**31 + 7, 2**32 - 1]
    case = Case(kind, 6, 2, 2, 64, 64, lib.HALVES, positions=positions)
    case.forward()
    case.check_forward()
    case.backward()
    case.check_backward()


def test_positions_are_the_tokens_where_none_are_given():
    case = Case(lib.F32, 5000, 1, 1, 16, 16, lib.HALVES, positions=np.arange(5000))
    case.shape.positions = None
    case.forward()
    case.check_forward()
    case.backward()
    case.check_backward()


@pytest.mark.parametrize("kind", KINDS)
def test_results_in_the_operands_place(kind):
    case = Case(kind, 33, 4, 2, 40, 20, lib.HALVES)
    lib.call("tc_rotary_norm", case.shape, *(h.ptr for h in case.held), *case.given, *(h.ptr for h in case.held))
    case.check_forward(case.held)
    for place in ("held_dz", "held"):
        case = Case(kind, 33, 4, 2, 40, 20, lib.HALVES)
        there = getattr(case, place)
        lib.call("tc_rotary_norm_backward", case.shape, *(d.ptr for d in case.held_dz), *(h.ptr for h in case.held),
                 *case.given, *(d.ptr for d in there), *(d.ptr for d in case.dw))
        case.check_backward(got=there)


def test_what_is_left_out():
    case = Case(lib.BF16, 9, 2, 2, 32, 32, lib.HALVES, weights=False)
    case.forward()
    case.check_forward()
    case.backward(dw=False)
    case.check_backward(dw=False)
    case = Case(lib.BF16, 9, 2, 2, 32, 32, lib.HALVES)
    lib.call("tc_rotary_norm_backward", case.shape, *(d.ptr for d in case.held_dz), *(h.ptr for h in case.held),
             *case.given, *(d.ptr for d in case.dx), None, case.dw[1].ptr)
    assert (case.dw[0].read() == 7).all()
    # Without a norm the operands are not read.
    case = Case(lib.F16, 9, 2, 2, 32, 32, lib.HALVES, normalize=False)
    lib.call("tc_rotary_norm_backward", case.shape, *(d.ptr for d in case.held_dz), None, None, None, None,
             *(d.ptr for d in case.dx), None, None)
    case.check_backward()


@pytest.mark.parametrize("pairs", [lib.HALVES, lib.NEIGHBOURS])
def test_elements_that_are_not_rotated_do_not_mix(pairs):
    case = Case(lib.F32, 3, 1, 1, 20, 6, pairs, normalize=False)
    case.x[0][1, 0, 9], case.x[0][1, 0, 19], case.x[0][2, 0, 12] = np.inf, np.nan, -np.inf
    case.held[0] = Heads(case.x[0], lib.F32)
    case.forward()
    got = case.out[0].read()
    assert np.array_equal(got[..., 6:], case.x[0][..., 6:], equal_nan=True)
    assert np.isfinite(got[..., :6]).all()


def test_the_weights_gradients_repeat_bit_for_bit():
    case = Case(lib.BF16, 9000, 4, 2, 64, 64, lib.HALVES, weight=lib.F32)
    case.backward()
    first = [d.read() for d in case.dw]
    case.backward()
    assert all(np.array_equal(a, d.read()) for a, d in zip(first, case.dw))
