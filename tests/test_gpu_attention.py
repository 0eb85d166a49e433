"""Causal attention over packed sequences and its gradients against the plain
forms in 64 bits.

Bounds: a weight p is off relatively by its score's error and a few roundings
of 32 bits, and by one rounding to the operands' type before its product; a
score by a rounding for each of its products' sums, of the sum of magnitudes.
With `loose` those 32-bit parts, a result sum_j p_j v_j is off by at most
(2 rounding + loose) sum_j p_j |v_j| and its own rounding; ds is off by that
of p (|do| . |v| + |do| . |o|), and the gradients by that weighted with |q| and
|k|."""

import numpy as np
import pytest

from tensorcrate_amd import lib
from tests import language
from tests.common import KIND_NAMES, KINDS, to_kind, widen
from tests.language import EPSILON_32, ROUNDING, TINY, near, stored

pytestmark = pytest.mark.gpu


class Heads:
    """[token, head, element] tensors side by side in one buffer, or heads
    before tokens, `shift` elements in; what lies around is `around`."""

    def __init__(self, tensors, kind, by_head=False, gap=0, shift=0, around=np.nan):
        self.kind, self.by_head, self.shift = kind, by_head, shift
        self.shapes = [t.shape for t in tensors]
        tokens, size = self.shapes[0][0], self.shapes[0][2]
        heads = sum(s[1] for s in self.shapes)
        whole = np.full((tokens, heads, size + gap), around)
        whole[:, :, :size] = np.concatenate(tensors, 1)
        if by_head:
            whole = whole.transpose(1, 0, 2)
        self.steps = (size + gap, tokens * (size + gap)) if by_head else (heads * (size + gap), size + gap)
        self.before = np.concatenate([np.full(shift, around), whole.reshape(-1), np.full(8, around)]).astype(np.float32)
        self.buffer = lib.Buffer.of(to_kind(self.before, kind))
        self.gap, self.heads, self.tokens, self.size = gap, heads, tokens, size

    @classmethod
    def like(cls, other):
        return cls([np.full(s, 7.0) for s in other.shapes], other.kind, other.by_head, other.gap, other.shift, 7.0)

    def ptr(self, n=0) -> int:
        skipped = sum(s[1] for s in self.shapes[:n])
        return self.buffer.ptr + (self.shift + skipped * self.steps[1]) * lib.DTYPE_SIZE[self.kind]

    def read(self):
        got = widen(self.kind, self.buffer.download(lib.NUMPY_TYPE[self.kind])).astype(np.float64)
        body = got[self.shift:got.size - 8].copy()
        shape = (self.heads, self.tokens) if self.by_head else (self.tokens, self.heads)
        body = body.reshape(*shape, self.size + self.gap)
        around = np.concatenate([got[:self.shift], got[got.size - 8:], body[..., self.size:].reshape(-1)])
        assert (around == 7.0).all(), "written outside the heads"
        if self.by_head:
            body = body.transpose(1, 0, 2)
        return np.split(body[..., :self.size], np.cumsum([s[1] for s in self.shapes])[:-1], 1)


def inputs(kind, tokens, heads, key_heads, size, seed, spread=1.0):
    rng = np.random.default_rng(seed)
    return [stored(rng.standard_normal((tokens, h, size)) * s, kind)
            for h, s in ((heads, spread), (key_heads, spread), (key_heads, 1.0), (heads, 1.0))]


def shape_of(kind, q, k, ends, scale, steps):
    tokens, heads, size = q.shape
    offsets = None if ends is None else lib.Buffer.of(np.array(ends, np.uint32))
    shape = lib.attention(kind, tokens, heads, k.shape[1], size, scale, None if offsets is None else offsets.ptr,
                          0 if ends is None else len(ends) - 1, *steps)
    return shape, offsets


def run(kind, q, k, v, d, ends, scale, layout="packed", keep=True):
    by_head, gap, shift = {"packed": (False, 0, 0), "heads": (True, 0, 0), "odd": (False, 3, 1)}[layout]
    if layout == "packed":
        whole = Heads([q, k, v], kind)
        at, steps = [whole.ptr(n) for n in range(3)], [whole.steps] * 3
        grads = Heads.like(whole)
        d_at = [grads.ptr(n) for n in range(3)]
    else:
        parts = [Heads([t], kind, by_head, gap, shift) for t in (q, k, v)]
        at, steps = [p.ptr() for p in parts], [p.steps for p in parts]
        grads = [Heads.like(p) for p in parts]
        d_at = [g.ptr() for g in grads]
    d_out = Heads([d], kind, by_head, gap, shift)
    out = Heads.like(d_out)
    shape, offsets = shape_of(kind, q, k, ends, scale, steps + [out.steps])
    normalizers = lib.Buffer(4 * q.shape[0] * q.shape[1])
    lib.call("tc_attention", shape, *at, out.ptr(), normalizers.ptr if keep else None)
    got = [out.read()[0]]
    if not keep:
        return got[0]
    got.append(normalizers.download(np.float32, q.shape[0] * q.shape[1]).reshape(q.shape[1], q.shape[0]).astype(np.float64))
    lib.call("tc_attention_backward", shape, d_out.ptr(), *at, out.ptr(), normalizers.ptr, *d_at)
    return got + (grads.read() if layout == "packed" else [g.read()[0] for g in grads])


def loose_of(q, k, scale):
    """The 32-bit error of a weight, relatively."""
    finite = lambda t: np.where(np.isfinite(t), t, 0.0)
    q, k = finite(q), finite(k)
    score = scale * np.sqrt((q * q).sum(2).max(initial=0) * (k * k).sum(2).max(initial=0))
    return EPSILON_32 * (64 + q.shape[0] / 8 + 2 * (q.shape[2] + 4) * score)


def check(kind, q, k, v, d, ends, scale, got):
    ends = [0, q.shape[0]] if ends is None else ends
    loose, u = loose_of(q, k, scale), ROUNDING[kind]
    out, normalizers, sizes = language.attention(q, k, v, ends, scale)
    near(got[0], out, (2 * u + loose) * sizes + u * np.abs(out) + TINY[kind], "out")
    finite = np.where(np.isfinite(normalizers), normalizers, 0.0)
    near(got[1], normalizers, loose + 4 * EPSILON_32 * np.abs(finite), "normalizers")
    grads, sizes = language.attention_backward(d, q, k, v, got[0], got[1], ends, scale)
    for name, have, want, size in zip(("dq", "dk", "dv"), got[2:], grads, sizes):
        # Weights from the normalizers as given: `loose` holds their rounding too.
        extra = 4 * EPSILON_32 * np.abs(finite).max(initial=0)
        near(have, want, (2 * u + 2 * loose + extra) * size + u * np.abs(want) + 2 * TINY[kind], name)


# Tokens, heads, key heads, head size, ends of sequences (None: all are one).
CASES = [
    (1, 1, 1, 1, None), (1, 8, 2, 64, None), (2, 2, 1, 3, None), (31, 1, 1, 32, None), (33, 2, 2, 33, None),
    (64, 3, 1, 40, None), (65, 2, 1, 64, None), (127, 4, 4, 80, None), (129, 2, 1, 96, None), (200, 4, 2, 100, None),
    (257, 2, 1, 128, None), (300, 7, 1, 16, None), (520, 1, 1, 127, None),
    (90, 2, 1, 24, [0, 1, 2, 3, 40, 40, 41, 90]), (190, 4, 2, 64, [3, 3, 70, 128, 129, 180]),
    (260, 2, 2, 128, [0, 64, 128, 192, 256]), (333, 6, 2, 72, [0, 32, 100, 333]), (140, 1, 1, 8, [0, 0, 0]),
    (400, 3, 3, 65, [100, 101, 231, 399]), (130, 2, 1, 48, list(range(131))),
    # Long sequences, whose blocks end with them, and so many that blocks do not.
    (1500, 2, 1, 64, [0, 1, 130, 700, 700, 1400]), (1100, 2, 2, 128, [50, 306, 562, 1090]),
    (520, 16, 4, 16, [0, 129, 400, 520]), (600, 4, 2, 40, [5] + list(range(9, 599, 4))),
    (300, 16, 4, 72, [0, 0, 0, 150, 151] + [290] * 40 + [291]), (700, 2, 1, 96, [0, 300] + [300] * 300 + [650]),
]


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:4])) + ("" if c[4] is None else f"-{len(c[4])}"))
def test_attention(kind, case):
    tokens, heads, key_heads, size, ends = case
    operands = inputs(kind, tokens, heads, key_heads, size, seed=tokens + size)
    scale = float(np.float32(size ** -0.5))
    for layout in ("packed", "heads", "odd"):
        check(kind, *operands, ends, scale, run(kind, *operands, ends, scale, layout))


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
def test_many_heads_share_a_key_head_and_large_scores(kind):
    for tokens, heads, key_heads, size, spread in ((150, 16, 1, 64, 1.0), (150, 12, 2, 128, 1.0), (140, 2, 1, 64, 4.0)):
        operands = inputs(kind, tokens, heads, key_heads, size, 3, spread)
        check(kind, *operands, None, 0.25, run(kind, *operands, None, 0.25))


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
def test_rising_scores(kind):
    # Each key scores above all before it: the running maximum moves on.
    tokens, size = 300, 32
    q, k, v, d = inputs(kind, tokens, 1, 1, size, 5)
    q[:] = 1.0
    k[:] = stored(np.arange(tokens) / 16, kind)[:, None, None]
    for scale in (0.02, 0.5):
        scale = float(np.float32(scale))
        check(kind, q, k, v, d, None, scale, run(kind, q, k, v, d, None, scale))


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("size", [64, 100])
@pytest.mark.parametrize("heads, empty", [(4, 0), (16, 40)])
def test_what_is_not_seen_does_not_matter(kind, value, size, heads, empty):
    # Tokens of no sequence, of one sequence only, and a late token, hold no
    # number: nothing that does not see them changes.
    # (Many sequences, most of them empty, have blocks across them.)
    ends = [2, 40, 90, 100, 230] + [300] * (1 + empty)
    q, k, v, d = inputs(kind, 310, heads, 2, size, 7)
    scale = float(np.float32(size ** -0.5))
    want = run(kind, q, k, v, d, ends, scale)
    for t in (q, k, v, d):
        t[:2] = t[300:] = value
        t[50:60] = value   # of the second sequence
        t[225] = value     # near the fourth's end
    got = run(kind, q, k, v, d, ends, scale)
    # Queries and what they write: their own sequence from the first such key on.
    forward = np.ones(310, bool)
    forward[50:90] = forward[225:230] = False
    for n in (0, 1):
        have, kept = (got[0], want[0]) if n == 0 else (got[1].T, want[1].T)
        assert np.array_equal(have[forward], kept[forward])
        assert not np.isfinite(have[50:60]).any() and not np.isfinite(have[225]).any()
    # Keys and values are seen by later queries of their sequence.
    backward = forward.copy()
    backward[40:90] = backward[100:230] = False
    assert np.array_equal(got[2][forward], want[2][forward])
    for n in (3, 4):
        assert np.array_equal(got[n][backward], want[n][backward])


def test_forward_alone_and_the_same_bits_again():
    operands = inputs(lib.BF16, 700, 8, 2, 64, 9)
    first, again = (run(lib.BF16, *operands, [0, 300, 700], 0.125) for _ in range(2))
    for a, b in zip(first, again):
        assert np.array_equal(a, b)
    assert np.array_equal(run(lib.BF16, *operands, [0, 300, 700], 0.125, keep=False), first[0])


def test_offsets_past_the_tokens_stay_within_them():
    # Offsets that are no order of these tokens answer something, from these tokens.
    operands = inputs(lib.F32, 70, 2, 1, 16, 11)
    for ends in ([0, 1000], [60, 2**32 - 1], [50, 20, 70], [2**32 - 1, 0, 5]):
        run(lib.F32, *operands, ends, 0.25)


def test_no_tokens():
    shape = lib.attention(lib.F32, 0, 2, 1, 16, 1.0, None, 0, *[(32, 16)] * 4)
    lib.call("tc_attention", shape, None, None, None, None, None)
    lib.call("tc_attention_backward", shape, *[None] * 9)


@pytest.mark.parametrize("kind", [lib.F16, lib.BF16], ids=KIND_NAMES.get)
@pytest.mark.parametrize("heads", [2, 16])
@pytest.mark.parametrize("length", [2, 5, 30, 200])
def test_short_sequences_lose_nothing_to_the_rounding_of_the_result(kind, heads, length):
    # Two roundings of independent values, of ds and of the result, are
    # 0.42 roundings each in the root of the mean square; what o lost as it was
    # rounded would be one more of up to a whole rounding.
    tokens = 1200 if length > 2 else 600
    ends = list(range(0, tokens + 1, length))
    q, k, v, d = inputs(kind, tokens, heads, 1, 64, length, 1.2)
    got = run(kind, q, k, v, d, ends, 0.125)
    out, normalizers, _ = language.attention(q, k, v, ends, 0.125)
    grads, _ = language.attention_backward(d, q, k, v, out, normalizers, ends, 0.125)
    for name, have, want in zip(("dq", "dk", "dv"), got[2:], grads):
        off = np.linalg.norm(have - want) / np.linalg.norm(want)
        assert off < 0.75 * ROUNDING[kind], (name, off / ROUNDING[kind])


LARGEST = {lib.F32: float(np.finfo(np.float32).max), lib.F16: 65504.0, lib.BF16: 3.3895313892515355e38}


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("size", [64, 100])
@pytest.mark.parametrize("heads, empty", [(4, 0), (16, 40)])
def test_numbers_that_are_not_seen_do_not_matter(kind, size, heads, empty):
    # The largest numbers in tokens of no sequence, and 2^13 times the usual
    # ones in another sequence, change no bit of what does not see them.
    ends = [2, 40, 90, 100, 230] + [300] * (1 + empty)
    operands = inputs(kind, 310, heads, 2, size, 13)
    scale = float(np.float32(size ** -0.5))
    want = run(kind, *operands, ends, scale)
    for sign in (1.0, -1.0):
        for t in operands:
            t[:2] = t[300:] = sign * LARGEST[kind]
        got = run(kind, *operands, ends, scale)
        for n, (have, kept) in enumerate(zip(got, want)):
            assert np.array_equal(have, kept), n
    for t in operands[2:]:  # values and the results' gradients
        t[100:230] *= 2.0**13
    got = run(kind, *operands, ends, scale)
    other = np.ones(310, bool)
    other[100:230] = False
    for n, (have, kept) in enumerate(zip(got, want)):
        if n == 1:
            have, kept = have.T, kept.T
        assert np.array_equal(have[other], kept[other]), n


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("heads", [2, 16])
def test_gradients_depend_on_what_they_sum_over_alone(kind, heads):
    # A query's gradient on the keys up to it, a key's on the queries from it on.
    tokens, at, size = 400, 150, 64
    q, k, v, d = inputs(kind, tokens, heads, 2, size, 17)
    want = run(kind, q, k, v, d, None, 0.125)
    for t in (k, v):
        t[at + 1:] *= 2.0**10
    got = run(kind, q, k, v, d, None, 0.125)
    assert np.array_equal(got[2][:at + 1], want[2][:at + 1])
    q, k, v, d = inputs(kind, tokens, heads, 2, size, 17)
    d[:at] *= 2.0**13
    got = run(kind, q, k, v, d, None, 0.125)
    for n in (3, 4):
        assert np.array_equal(got[n][at:], want[n][at:])


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("heads", [2, 16])
@pytest.mark.parametrize("where", ["first", "last", "rising", "falling"])
def test_gradients_of_rows_of_very_different_magnitudes(kind, heads, where):
    tokens, size = 300, 64
    q, k, v, d = inputs(kind, tokens, heads, 2, size, 19)
    at = np.arange(tokens)
    power = {"first": np.where(at == 0, 11, -8), "last": np.where(at == tokens - 1, 11, -8), "rising": at // 16 - 8,
             "falling": 10 - at // 16}[where]
    d *= 2.0 ** power.astype(float)[:, None, None]
    for ends in (None, [0, 150, 300]):
        check(kind, q, k, v, d, ends, 0.125, run(kind, q, k, v, d, ends, 0.125))


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("heads", [1, 8])
def test_a_query_whose_scores_are_all_minus_infinity(kind, heads):
    # 0 / 0 of the definition, not the zeros of a token in no sequence; and a
    # key of that score beside others has the weight 0.
    q, k, v, d = inputs(kind, 200, heads, 1, 64, 21)
    q[:] = np.abs(q) + 0.5
    k[50] = -np.inf
    for ends in ([10, 50, 190], [10, 50] + [190] * 120):
        got = run(kind, q, k, v, d, ends, 0.125)
        assert np.isnan(got[0][50]).all() and np.isneginf(got[1][:, 50]).all()
        assert np.isfinite(got[0][:50]).all() and np.isfinite(got[0][51:]).all()
        assert not got[0][:10].any() and not got[0][190:].any()
        assert np.isfinite(got[1][:, 51:190]).all() and np.isneginf(got[1][:, 190:]).all()


def test_more_than_2_31_sequences():
    # All but the last few of them empty.
    count, ends = 2**31 + 1000, [0, 30, 30, 101, 190]
    q, k, v, d = inputs(lib.F32, 200, 1, 1, 16, 23)
    want = run(lib.F32, q, k, v, d, ends, 0.25)
    zero, last = np.zeros(1, np.uint32), np.array(ends, np.uint32)
    offsets = lib.Buffer(4 * (count + 1))
    lib.call("tc_fill", offsets.ptr, count + 1, 4, zero.ctypes.data)
    lib.call("tc_upload", offsets.ptr + 4 * (count + 1 - last.size), last.ctypes.data, last.nbytes)
    parts = [Heads([t], lib.F32) for t in (q, k, v, d)]
    out, *grads = [Heads.like(p) for p in (parts[3], *parts[:3])]
    at = [p.ptr() for p in parts]
    shape = lib.attention(lib.F32, 200, 1, 1, 16, 0.25, offsets.ptr, count, *[p.steps for p in parts])
    normalizers = lib.Buffer(4 * 200)
    lib.call("tc_attention", shape, *at[:3], out.ptr(), normalizers.ptr)
    lib.call("tc_attention_backward", shape, at[3], *at[:3], out.ptr(), normalizers.ptr, *[g.ptr() for g in grads])
    have = [out.read()[0], normalizers.download(np.float32, 200)[None].astype(np.float64)] + [g.read()[0] for g in grads]
    ends = [0, 30, 101, 190]
    check(lib.F32, q, k, v, d, ends, 0.25, have)
    check(lib.F32, q, k, v, d, ends, 0.25, want)
