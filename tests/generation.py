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


# ---- a cache of keys and values ---------------------------------------------

NO_PAGE = 0xFFFFFFFF


def quantised(x):
    """(whole numbers, scales) of the rows x, in 32 bits as an IEEE machine
    computes them."""
    x = np.asarray(x, np.float32)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        most = np.abs(x).max(-1)
        finite = np.isfinite(most)
        scales = np.where(finite, (most / np.float32(127)).astype(np.float32), np.float32(np.nan)).astype(np.float32)
        q = np.clip(np.rint(x / scales[..., None]), -127, 127)
    q = np.where((finite & (scales > 0))[..., None], q, 0)
    return q.astype(np.int8), scales


class World:
    """A cache on the host and on the device, with sequences of `lengths`
    tokens of which the last `new` are a call's, `lead` tokens in no sequence
    before them and `trail` behind.  Nothing is in the cache, only poison:
    0xff in every byte, a NaN in every type but the 8-bit numbers."""

    def __init__(self, kind, fmt, key_heads, size, page, lengths, new=None, prefix=0, lead=0, trail=0, extra=1, seed=0):
        rng = np.random.default_rng(seed)
        self.kind, self.fmt, self.key_heads, self.size, self.page = kind, fmt, key_heads, size, page
        self.lengths, self.prefix = list(lengths), prefix
        self.new = [1] * len(self.lengths) if new is None else list(new)
        per = 16 if fmt == lib.CACHE_INT8 else 16 // lib.DTYPE_SIZE[kind]
        self.row = -(-size // per) * per
        pages = [-(-n // page) for n in self.lengths]
        prefix_pages = -(-prefix // page)
        self.page_count = prefix_pages + sum(pages) + 2
        order = rng.permutation(self.page_count).astype(np.uint32)
        self.prefix_pages, at = order[:prefix_pages], prefix_pages
        self.most = max(pages, default=0) + extra
        self.table = np.full((len(pages), self.most), NO_PAGE, np.uint32)
        for s, n in enumerate(pages):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.offsets = None if new is None and not lead and not trail else (
            lead + np.concatenate([[0], np.cumsum(self.new)])).astype(np.uint32)
        self.lead, self.tokens = lead, lead + sum(self.new) + trail
        self.entry = np.int8 if fmt == lib.CACHE_INT8 else lib.NUMPY_TYPE[kind]
        shape = (self.page_count, key_heads, page, self.row)
        self.pools = [np.full(int(np.prod(shape)) * np.dtype(self.entry).itemsize, 0xFF, np.uint8).view(
            self.entry).reshape(shape) for _ in range(2)]
        self.scales = [np.full(shape[:-1], np.nan, np.float32) for _ in range(2)]
        self.device = None

    def upload(self):
        """The host's cache to the device, and the structs of the calls."""
        quant = self.fmt == lib.CACHE_INT8
        self.device = [lib.Buffer.of(p) for p in self.pools] + [lib.Buffer.of(s) if quant else None for s in self.scales]
        self.tables = [None if a is None else lib.Buffer.of(np.ascontiguousarray(a, np.uint32)) for a in (
            self.offsets, np.array(self.lengths), self.table, self.prefix_pages)]
        at = lambda b: None if b is None else b.ptr
        self.cache = lib.cache(self.kind, self.fmt, self.key_heads, self.size, self.page, self.page_count,
                               *map(at, self.device))
        offsets, lengths, table, prefix = map(at, self.tables)
        self.batch = lib.cache_batch(self.tokens, len(self.lengths), offsets, lengths, table, self.most, self.prefix,
                                     prefix if self.prefix else None)

    def download(self):
        quant = self.fmt == lib.CACHE_INT8
        pools = [b.download(self.entry).reshape(p.shape) for b, p in zip(self.device[:2], self.pools)]
        scales = [b.download(np.float32).reshape(s.shape) if quant else s for b, s in zip(self.device[2:], self.scales)]
        return pools, scales

    def places(self):
        """(token, sequence, position) of each token in a sequence."""
        at = self.lead
        for s, n in enumerate(self.new):
            for i in range(n):
                yield at + i, s, self.lengths[s] - n + i
            at += n

    def slot(self, pages, position):
        """(page, slot), or None."""
        if position < 0 or position >= len(pages) * self.page:
            return None
        page = int(pages[position // self.page])
        return (page, position % self.page) if page < self.page_count else None

    def put(self, place, n, rows):
        """The heads `rows` [key head, element] of a token into pool n."""
        if place is None:
            return
        page, slot = place
        self.pools[n][page, :, slot] = 0
        if self.fmt == lib.CACHE_INT8:
            q, scales = quantised(rows)
            self.pools[n][page, :, slot, :self.size] = q
            self.scales[n][page, :, slot] = scales
        else:
            self.pools[n][page, :, slot, :self.size] = to_kind(np.asarray(rows, np.float32), self.kind)

    def get(self, place, n, head):
        """A row of pool n as the numbers it stands for, in 64 bits."""
        if place is None:
            return np.zeros(self.size)
        page, slot = place
        row = self.pools[n][page, head, slot, :self.size]
        if self.fmt == lib.CACHE_INT8:
            with np.errstate(invalid="ignore"):
                return row.astype(np.float64) * np.float64(self.scales[n][page, head, slot])
        return widen(self.kind, row).astype(np.float64)

    def fill(self, rng, spread=1.0):
        """Normal keys and values for all sequences and the prefix."""
        for pages, count in [(self.prefix_pages, self.prefix)] + list(zip(self.table, self.lengths)):
            for position in range(count):
                for n in range(2):
                    self.put(self.slot(pages, position), n,
                             rng.standard_normal((self.key_heads, self.size)) * (spread if n == 0 else 1.0))

    def rows(self, n, head, sequence):
        """Pool n's rows of the prefix and of a sequence."""
        length = min(self.lengths[sequence], self.most * self.page)
        out = [self.get(self.slot(self.prefix_pages, p), n, head) for p in range(self.prefix)]
        out += [self.get(self.slot(self.table[sequence], p), n, head) for p in range(length)]
        return np.array(out).reshape(-1, self.size)


def cache_attention(world, q, scale):
    """(out, normalizers, sum of p |v|) of the queries [token, head, element]
    over the cache; what a query does not see is not touched."""
    tokens, heads, size = q.shape
    group = heads // world.key_heads
    out, sizes = np.zeros_like(q), np.zeros_like(q)
    normalizers = np.full((heads, tokens), -np.inf)
    held = {}
    for token, s, position in world.places():
        for head in range(heads):
            key = (s, head // group)
            if key not in held:
                held[key] = [world.rows(n, head // group, s) for n in range(2)]
            k, v = held[key]
            seen = max(0, min(world.prefix + position + 1, len(k)))
            if not seen:
                continue
            with np.errstate(invalid="ignore", over="ignore"):
                scores = scale * (k[:seen] @ q[token, head])
                most = scores.max()
                e = np.exp(scores - most)
                p = e / e.sum()
                out[token, head] = p @ v[:seen]
                sizes[token, head] = p @ np.abs(v[:seen])
                normalizers[head, token] = most + np.log(e.sum())
    return out, normalizers, sizes
