"""Attention over a cache against the plain form in 64 bits.

Bounds: a weight is off relatively by its score's error and a few roundings of
32 bits (`loose`), and by its rounding before the product with the values: none
in f32, one of f16 in f16 and over 8 bits, in bf16 one of 16 bits (two parts of
bf16's 8).  As f16 weights are rounded times 2^6 where the largest is at least 1,
so that one is off by at most 2^-31 besides, of a sum of 1 or more; over 8 bits
they are weights times a scale, against a power of two at most 16 times the
largest scale: 2^-27 of that."""

import numpy as np
import pytest

from tensorcrate_amd import lib
from tests import generation
from tests.common import KIND_NAMES, KINDS
from tests.generation import NO_PAGE, Heads, World
from tests.language import EPSILON_32, ROUNDING, TINY, near, stored

pytestmark = pytest.mark.gpu

FORMATS = [lib.CACHE_PLAIN, lib.CACHE_INT8]


def run(world, q, scale, layout={}, keep=True):
    held = Heads(q, world.kind, **layout)
    out = Heads.empty(*q.shape, world.kind, **layout)
    normalizers = lib.Buffer.of(np.full(q.shape[0] * q.shape[1], 7.0, np.float32))
    lib.call("tc_cache_attention", world.cache, world.batch, q.shape[1], scale, held.ptr, *held.steps, out.ptr, *out.steps,
             normalizers.ptr if keep else None)
    return out.read(), normalizers.download(np.float32).reshape(q.shape[1], q.shape[0]).astype(np.float64)


def check(world, q, scale, got):
    out, normalizers, sizes = generation.cache_attention(world, q, scale)
    rows = [world.rows(n, h, s) for n in range(2) for h in range(world.key_heads) for s in range(len(world.lengths))]
    finite = lambda t: np.where(np.isfinite(t), t, 0.0)
    longest = lambda rows: max((np.sqrt((finite(r) ** 2).sum(1)).max(initial=0) for r in rows), default=0.0)
    score = scale * longest(rows[:len(rows) // 2]) * np.sqrt((finite(q) ** 2).sum(2)).max(initial=0)
    keys = max((len(r) for r in rows), default=0)
    loose = EPSILON_32 * (64 + keys / 8 + 2 * (world.size + 6) * score)
    quant = world.fmt == lib.CACHE_INT8
    f16 = world.kind == lib.F16 or (quant and world.kind == lib.BF16)
    weight = 2.0**-11 if f16 else 0.0 if world.kind == lib.F32 else 2.0**-16
    # Over 8 bits every value counts as the largest one of all.
    far = 0.0
    for r in rows[len(rows) // 2:] if f16 else []:
        far += 2.0**-27 * len(r) * np.abs(finite(r)).max(initial=0) if quant else 2.0**-31 * np.abs(finite(r)).sum(0).max(initial=0)
    near(got[0], out, (weight + loose) * sizes + far + ROUNDING[world.kind] * np.abs(out) + TINY[world.kind], "out")
    near(got[1], normalizers, loose + 4 * EPSILON_32 * np.abs(finite(normalizers)), "normalizers")


def queries(world, heads, seed=0, spread=1.0):
    return stored(np.random.default_rng(seed).standard_normal((world.tokens, heads, world.size)) * spread, world.kind)


def both(world, heads, seed=0, layout={}, spread=1.0):
    world.fill(np.random.default_rng(seed + 1), spread)
    world.upload()
    q = queries(world, heads, seed, spread)
    scale = float(np.float32(world.size ** -0.5))
    check(world, q, scale, run(world, q, scale, layout))
    return q, scale


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("size", [1, 8, 31, 32, 33, 40, 64, 75, 80, 96, 100, 127, 128])
def test_sizes(kind, fmt, size):
    both(World(kind, fmt, 2, size, 16, [1, 15, 16, 17, 33, 70, 129, 300]), 6)


# Key heads, query heads, page, lengths, new tokens, prefix, tokens in no
# sequence before and behind.
CASES = {
    "one key": (1, 1, 4, [1], None, 0, 0, 0),
    "one sequence": (2, 8, 16, [1000], None, 0, 0, 0),
    "pages of one": (1, 3, 1, [150, 40], None, 0, 0, 0),
    "odd pages": (3, 3, 7, [5, 64, 200, 129], None, 0, 0, 0),
    "long pages": (1, 2, 500, [499, 500, 501], None, 0, 0, 0),
    "many heads share": (1, 40, 16, [90, 300], None, 0, 0, 0),
    "many sequences": (1, 2, 8, [1 + 3 * n % 61 for n in range(600)], None, 0, 0, 0),
    "drafts": (2, 4, 16, [5, 40, 300, 129], [5, 3, 6, 4], 0, 0, 0),
    "drafts on tile borders": (1, 4, 16, [34, 66, 130, 257], [4, 4, 4, 8], 0, 0, 0),
    "a prompt": (2, 4, 16, [200], [200], 0, 0, 0),
    "prompts and tokens": (1, 2, 16, [130, 1, 60, 500], [130, 1, 10, 1], 0, 0, 0),
    "around": (2, 2, 16, [30, 40], [3, 2], 0, 4, 5),
    "empty sequences": (1, 2, 16, [30, 9, 40, 0], [2, 0, 1, 0], 0, 0, 0),
    "nothing cached": (1, 2, 16, [0, 0], None, 0, 0, 0),
    "more tokens than keys": (1, 2, 16, [2, 50], [5, 2], 0, 0, 0),
    "prefix": (2, 8, 16, [1, 30, 200, 7], None, 300, 0, 0),
    "prefix of one": (1, 2, 16, [1, 30], None, 1, 0, 0),
    "prefix on odd pages": (1, 4, 10, [17, 3], [3, 1], 123, 0, 0),
    "prefix and nothing": (1, 2, 16, [0, 5], None, 64, 0, 0),
    "prefix and tokens in it": (1, 2, 16, [2, 50], [5, 2], 40, 0, 0),
    "prefix and many": (1, 8, 16, [1 + n % 9 for n in range(70)], None, 700, 0, 0),
    "prefix around": (1, 2, 16, [30, 9], [2, 1], 50, 2, 3),
    "long": (1, 2, 64, [6000, 100], None, 0, 0, 0),
}


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("name", CASES)
def test_batches(kind, fmt, name):
    key_heads, heads, page, lengths, new, prefix, lead, trail = CASES[name]
    layout = dict(gap=3, token_gap=5, shift=1) if len(name) % 2 else dict(turned=True)
    both(World(kind, fmt, key_heads, 40, page, lengths, new, prefix, lead, trail), heads, len(name), layout)


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("fmt", FORMATS)
def test_wide_heads(kind, fmt):
    both(World(kind, fmt, 2, 128, 16, [700, 90, 33], prefix=200), 8)
    both(World(kind, fmt, 1, 128, 64, [700, 90], [9, 3]), 4)
    both(World(kind, fmt, 1, 96, 64, [700, 90], [9, 3], prefix=90), 4)


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("fmt", FORMATS)
def test_large_scores(kind, fmt):
    # Weights of which a few are all: the running maximum moves.
    both(World(kind, fmt, 1, 64, 16, [400, 90]), 4,
         spread=4.0)


@pytest.mark.parametrize("fmt", FORMATS)
def test_pages_that_are_none(fmt):
    world = World(lib.F32, fmt, 1, 24, 8, [40, 30, 20], prefix=30)
    world.table[0, 2], world.table[2, 0] = world.page_count, NO_PAGE
    world.prefix_pages[1] = NO_PAGE
    both(world, 2)
    # A length past the sequence's pages, and past the table; and past what is
    # written too, which is seen then.
    for lengths in ([40, 32, 24], [40, 30, 20]):
        world = World(lib.F32, fmt, 1, 24, 8, lengths)
        world.fill(np.random.default_rng(1))
        world.lengths = [40, 37, 400]
        world.upload()
        q = queries(world, 2)
        got = run(world, q, 0.2)
        assert np.isfinite(got[0]).all() == (lengths[1] == 32)
        check(world, q, 0.2, got)


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
def test_what_later_tokens_hold(kind, fmt, what):
    # Keys and values of a sequence's last tokens, which earlier ones do not see.
    for lengths, new, prefix in (([70, 40], [4, 3], 0), ([33, 200], [3, 8], 50)):
        world = World(kind, fmt, 1, 40, 16, lengths, new, prefix)
        rng = np.random.default_rng(3)
        world.fill(rng)
        for s, n in enumerate(lengths):
            place = world.slot(world.table[s], n - 1)
            for pool in range(2):
                rows = rng.standard_normal((1, 40))
                rows[0, 5 + pool] = what
                world.put(place, pool, rows)
            world.put(world.slot(world.table[s], n - 2), 1, np.where(np.arange(40) == 9, what, rng.standard_normal((1, 40))))
        world.upload()
        q = queries(world, 2)
        got = run(world, q, 0.2)
        out, normalizers, _ = generation.cache_attention(world, q, 0.2)
        # Rows that see none of it are as always; of those that do, the elements
        # and kinds of what they see.
        assert np.isfinite(out[0]).all() and not np.isfinite(out[new[0] - 1]).all()
        check(world, q, 0.2, got)


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
def test_scores_of_minus_infinity(kind):
    world = World(kind, lib.CACHE_PLAIN, 1, 16, 16, [40, 5, 3], prefix=0)
    rng = np.random.default_rng(3)
    world.fill(rng)
    for s, n in ((1, 5), (0, 30)):
        for position in range(n):
            rows = rng.standard_normal((1, 16))
            rows[0, 0] = -np.inf
            world.put(world.slot(world.table[s], position), 0, rows)
    world.upload()
    q = np.abs(queries(world, 1)) + 0.5
    q = stored(q, kind)
    got = run(world, q, 0.2)
    assert np.isnan(got[0][1]).all() and got[1][0, 1] == -np.inf
    out, normalizers, _ = generation.cache_attention(world, q, 0.2)
    normalizers[0, 1] = -np.inf
    assert np.isfinite(got[0][[0, 2]]).all() and np.isfinite(got[1][0, [0, 2]]).all()
    assert np.abs(got[0][[0, 2]] - out[[0, 2]]).max() < 0.05


def test_without_normalizers_and_repeated():
    world = World(lib.BF16, lib.CACHE_INT8, 2, 64, 16, [500, 30, 2000], prefix=100)
    q, scale = both(world, 4)
    first, _ = run(world, q, scale)
    again, left = run(world, q, scale, keep=False)
    assert np.array_equal(first, again) and (left == 7).all()


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
def test_as_attention_over_the_same_keys(kind):
    # A prompt's attention, and the same tokens over a cache of their keys.
    from tests import language
    rng = np.random.default_rng(0)
    tokens, heads, key_heads, size = 150, 4, 2, 64
    q, k, v = (stored(rng.standard_normal((tokens, h, size)), kind) for h in (heads, key_heads, key_heads))
    held = [Heads(t, kind) for t in (q, k, v)]
    out = Heads.empty(tokens, heads, size, kind)
    shape = lib.attention(kind, tokens, heads, key_heads, size, 0.125, None, 0, *(h.steps for h in held), out.steps)
    lib.call("tc_attention", shape, *(h.ptr for h in held), out.ptr, None)
    world = World(kind, lib.CACHE_PLAIN, key_heads, size, 16, [tokens], [tokens])
    world.upload()
    lib.call("tc_cache_write", world.cache, world.batch, held[1].ptr, *held[1].steps, held[2].ptr, *held[2].steps)
    got, _ = run(world, q, 0.125)
    want, _, sizes = language.attention(q, k, v, [0, tokens], 0.125)
    bound = 4 * ROUNDING[kind] * sizes + 1e-5
    near(out.read(), want, bound, "attention")
    near(got, want, bound, "over the cache")
