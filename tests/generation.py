"""Plain implementations of the operators of generation in 64 bits, written
from their formulas, and what the tests of them share."""

from __future__ import annotations

import numpy as np

from tensorcrate_amd import lib
from tests.common import to_kind, widen


class Heads:
    """[token][head][element] of one kind on the device: `gap` elements behind
    each head, `token_gap` behind each token and `shift` before the first, all
    of it filled with `around`.  With `turned`, heads lie further apart than
    tokens."""

    def __init__(self, values, kind, gap=0, token_gap=0, shift=0, around=np.nan, turned=False):
        values = np.asarray(values, np.float32)
        self.tokens, self.heads, self.size = values.shape
        self.kind, self.shift = kind, shift
        if turned:
            self.token_step = self.size + gap
            self.head_step = self.tokens * self.token_step + token_gap
            count = self.heads * self.head_step
        else:
            self.head_step = self.size + gap
            self.token_step = self.heads * self.head_step + token_gap
            count = self.tokens * self.token_step
        self.places = (shift + np.arange(self.tokens)[:, None, None] * self.token_step
                       + np.arange(self.heads)[:, None] * self.head_step + np.arange(self.size))
        self.whole = np.full(shift + count + 8, around, np.float32)
        self.whole[self.places] = values
        self.buffer = lib.Buffer.of(to_kind(self.whole, kind))

    @classmethod
    def empty(cls, tokens, heads, size, kind, **layout):
        return cls(np.full((tokens, heads, size), 7.0), kind, around=7.0, **layout)

    @property
    def ptr(self) -> int:
        return self.buffer.ptr + self.shift * lib.DTYPE_SIZE[self.kind]

    @property
    def steps(self) -> tuple[int, int]:
        return self.token_step, self.head_step

    def read(self) -> np.ndarray:
        """The heads; what lies around them has to be as it was."""
        got = widen(self.kind, self.buffer.download(lib.NUMPY_TYPE[self.kind]))
        outside = np.ones(got.size, bool)
        outside[self.places] = False
        before = widen(self.kind, to_kind(self.whole, self.kind))
        assert np.array_equal(got[outside], before[outside], equal_nan=True), "written outside the heads"
        return got[self.places].astype(np.float64)


# ---- rotary positions -------------------------------------------------------


def pairs_of(size, rotary, pairs):
    """(first, second) elements of the rotated pairs."""
    i = np.arange(rotary // 2)
    return (i, i + rotary // 2) if pairs == lib.HALVES else (2 * i, 2 * i + 1)


def turned(y, positions, frequencies, pairs, back=False):
    """The heads y [token, head, element] turned, and for each element the sum
    of the magnitudes that its result is made of."""
    angles = positions.astype(np.float64)[:, None] * frequencies.astype(np.float64)
    cos, sin = np.cos(angles)[:, None], np.sin(angles)[:, None] * (-1 if back else 1)
    a, b = pairs_of(y.shape[2], 2 * len(frequencies), pairs)
    z, loose = y.copy(), np.abs(y)
    if len(frequencies):
        z[..., a] = y[..., a] * cos - y[..., b] * sin
        z[..., b] = y[..., b] * cos + y[..., a] * sin
        loose[..., a] = loose[..., b] = np.abs(y[..., a]) + np.abs(y[..., b])
    return z, loose


def rotary(x, weight, epsilon, positions, frequencies, pairs):
    """(z, magnitudes) of the heads x; with `epsilon` None there is no norm."""
    y = x
    if epsilon is not None:
        y = x / np.sqrt((x ** 2).mean(2, keepdims=True) + epsilon) * weight
    return turned(y, positions, frequencies, pairs)


def rotary_backward(dz, x, weight, epsilon, positions, frequencies, pairs):
    """((dx, dw), the sums of magnitudes that their errors go by)."""
    dy, loose = turned(dz, positions, frequencies, pairs, back=True)
    if epsilon is None:
        return (dy, None), (loose, None)
    scale = 1 / np.sqrt((x ** 2).mean(2, keepdims=True) + epsilon)
    u, g = x * scale, dy * weight
    dx = scale * (g - u * (g * u).mean(2, keepdims=True))
    sizes = scale * np.abs(weight) * loose + scale * np.abs(u) * (np.abs(weight * u) * loose).mean(2, keepdims=True)
    return (dx, (dy * u).sum((0, 1))), (sizes, (loose * np.abs(u)).sum((0, 1)))
