"""Plain implementations of the language-model operators in 64 bits, written
from their formulas, and what the tests of them share."""

from __future__ import annotations

import numpy as np

from tensorcrate_amd import lib
from tests.common import to_kind, widen

# The relative rounding of one result to its type.
ROUNDING = {lib.F32: 2.0**-24, lib.F16: 2.0**-11, lib.BF16: 2.0**-8}
# The smallest steps of a type around zero, half of them a rounding's error.
TINY = {lib.F32: 2.0**-149, lib.F16: 2.0**-25, lib.BF16: 2.0**-134}
EPSILON_32 = 2.0**-24


def stored(values, kind) -> np.ndarray:
    """`values` as `kind` holds them, in 64 bits."""
    return widen(kind, to_kind(np.asarray(values, np.float32), kind)).astype(np.float64)


class Rows:
    """Rows of one kind on the device, `gap` elements between them and `shift`
    elements before the first, all of it filled with `around`."""

    def __init__(self, values, kind, gap=0, shift=0, around=np.nan):
        values = np.asarray(values, np.float32)
        self.rows, self.cols = values.shape
        self.kind, self.step, self.shift = kind, self.cols + gap, shift
        self.whole = np.full(shift + self.rows * self.step + 8, around, np.float32)
        for row in range(self.rows):
            at = shift + row * self.step
            self.whole[at:at + self.cols] = values[row]
        self.buffer = lib.Buffer.of(to_kind(self.whole, kind))

    @classmethod
    def empty(cls, rows, cols, kind, gap=0, shift=0):
        return cls(np.full((rows, cols), 7.0), kind, gap, shift, around=7.0)

    @property
    def ptr(self) -> int:
        return self.buffer.ptr + self.shift * lib.DTYPE_SIZE[self.kind]

    def read(self) -> np.ndarray:
        """The rows; what lies around them has to be as it was."""
        got = widen(self.kind, self.buffer.download(lib.NUMPY_TYPE[self.kind]))
        inside = np.zeros(got.size, bool)
        out = np.empty((self.rows, self.cols), np.float64)
        for row in range(self.rows):
            at = self.shift + row * self.step
            inside[at:at + self.cols] = True
            out[row] = got[at:at + self.cols]
        before = widen(self.kind, to_kind(self.whole, self.kind))
        assert np.array_equal(got[~inside], before[~inside], equal_nan=True), "written outside the rows"
        return out


def near(got, want, bound, what: str) -> None:
    """Every value within its own bound; infinities and NaNs where they are wanted."""
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, what
    special = ~np.isfinite(want)
    assert np.array_equal(got[special], want[special], equal_nan=True), what
    with np.errstate(invalid="ignore"):
        off = np.abs(got - want)[~special]
    most = np.broadcast_to(np.asarray(bound, np.float64), want.shape)[~special]
    bad = ~(off <= most)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, by up to {np.nanmax(off[bad] / np.maximum(most[bad], 1e-300)):.3g} bounds"


# ---- layer norm -------------------------------------------------------------


def layer_norm(x, weight, bias, epsilon):
    mean = x.mean(1, keepdims=True)
    scale = 1.0 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + epsilon)
    return (x - mean) * scale * weight + bias, mean[:, 0], scale[:, 0]


def layer_norm_backward(dy, x, weight, mean, scale):
    u = (x - mean[:, None]) * scale[:, None]
    g = dy * weight
    dx = scale[:, None] * (g - g.mean(1, keepdims=True) - u * (g * u).mean(1, keepdims=True))
    return dx, (dy * u).sum(0), dy.sum(0)


# ---- log probabilities ------------------------------------------------------


def log_probabilities(x, tokens, top):
    """(log p of the tokens, normalizers, entropies, top log p, top tokens)."""
    rows, cols = x.shape
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        most = x.max(1, keepdims=True)
        shift = np.where(most == -np.inf, 0.0, most)
        total = np.exp(x - shift).sum(1, keepdims=True)
        normalizers = (shift + np.log(total))[:, 0]
        log_p = np.where(most == -np.inf, -np.inf, x - normalizers[:, None])
        p = np.exp(log_p)
        entropies = -np.where(p == 0, 0.0, p * log_p).sum(1) + 0.0
    given = np.array([log_p[r, t] if t < cols else 0.0 for r, t in enumerate(tokens)])
    # Highest first, a NaN last, equal logits by the lower token.
    order = np.lexsort((np.arange(cols)[None].repeat(rows, 0), -np.where(np.isnan(x), -np.inf, x), np.isnan(x)))
    picked = order[:, :top]
    return given, normalizers, entropies, np.take_along_axis(log_p, picked, 1), picked


def log_probabilities_backward(x, tokens, normalizers, entropies, d_given, d_entropies):
    d = np.zeros_like(x)
    for r, t in enumerate(tokens):
        g = d_given[r] if t < x.shape[1] else 0.0
        h = d_entropies[r]
        if (g == 0 and h == 0) or normalizers[r] == -np.inf:
            continue
        log_p = x[r] - normalizers[r]
        p = np.exp(log_p)
        with np.errstate(invalid="ignore"):
            d[r] = -np.where(p == 0, 0.0, p * (g + h * (log_p + entropies[r])))
        if t < x.shape[1]:
            d[r, t] += g
    return d


# ---- attention --------------------------------------------------------------


def attention(q, k, v, ends, scale):
    """(out, normalizers, sum of p |v|) of queries [token, head, element] and
    keys and values [token, key head, element], sequences ending at `ends`
    (the first at ends[0] begins the first); what a query does not see is not
    touched."""
    tokens, heads, size = q.shape
    group = heads // k.shape[1]
    out, sizes = np.zeros_like(q), np.zeros_like(q)
    normalizers = np.full((heads, tokens), -np.inf)
    for begin, end in zip(ends, ends[1:]):
        for head in range(heads):
            h = head // group
            for row in range(begin, end):
                seen = slice(begin, row + 1)
                with np.errstate(invalid="ignore", over="ignore"):
                    scores = scale * (k[seen, h] @ q[row, head])
                    most = scores.max()
                    e = np.exp(scores - most)
                    p = e / e.sum()
                    out[row, head] = p @ v[seen, h]
                    sizes[row, head] = p @ np.abs(v[seen, h])
                    normalizers[head, row] = most + np.log(e.sum())
    return out, normalizers, sizes


def attention_backward(d, q, k, v, out, normalizers, ends, scale):
    """((dq, dk, dv), the sums of magnitudes that their errors go by)."""
    tokens, heads, size = q.shape
    group = heads // k.shape[1]
    grads = [np.zeros_like(t) for t in (q, k, v)]
    sizes = [np.zeros_like(t) for t in (q, k, v)]
    for begin, end in zip(ends, ends[1:]):
        for head in range(heads):
            h = head // group
            for row in range(begin, end):
                seen = slice(begin, row + 1)
                with np.errstate(invalid="ignore", over="ignore"):
                    p = np.exp(scale * (k[seen, h] @ q[row, head]) - normalizers[head, row])
                    dot = d[row, head] @ out[row, head]
                    ds = p * (v[seen, h] @ d[row, head] - dot)
                    loose = p * (np.abs(v[seen, h]) @ np.abs(d[row, head]) + np.abs(d[row, head]) @ np.abs(out[row, head]))
                    grads[0][row, head] = scale * (ds @ k[seen, h])
                    grads[1][seen, h] += scale * np.outer(ds, q[row, head])
                    grads[2][seen, h] += np.outer(p, d[row, head])
                    sizes[0][row, head] = scale * (loose @ np.abs(k[seen, h]))
                    sizes[1][seen, h] += scale * np.outer(loose, np.abs(q[row, head]))
                    sizes[2][seen, h] += np.outer(p, np.abs(d[row, head]))
    return grads, sizes
