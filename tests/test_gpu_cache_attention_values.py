"""Attention over a cache where rows differ widely: what one row holds may not
cost another's precision.

Every bound here goes by what the query itself sees: by the sum of p |v| of each
element.  A weight is off relatively by its score's error and some roundings of
32 bits (`loose`, as in test_gpu_cache_attention.py), and by its own rounding
for the product with the values: none in f32, 2^-16 in two parts of bf16 (two
roundings of 2^-8), 2^-21 in two of f16 (the first cut off, which leaves less
than 2^-10, and that rounded by 2^-11), which, rounded times 2^6 where the largest
is at least 1, are off by at most 2^-31 besides."""

import numpy as np
import pytest

from tensorcrate_amd import lib
from tests import generation
from tests.common import KIND_NAMES, KINDS
from tests.generation import World
from tests.language import EPSILON_32, ROUNDING, TINY, near
from tests.test_gpu_cache_attention import check as attention_check
from tests.test_gpu_cache_attention import queries, run

pytestmark = pytest.mark.gpu

SIZE, SCALE = 40, 0.2
WEIGHT = {lib.F32: 0.0, lib.F16: 2.0**-21, lib.BF16: 2.0**-16}  # of two parts


def check(world, q, got, weight, far=0.0):
    out, normalizers, sizes = generation.cache_attention(world, q, SCALE)
    keys = [world.rows(0, h, s) for h in range(world.key_heads) for s in range(len(world.lengths))]
    score = SCALE * max(np.sqrt((k ** 2).sum(1)).max(initial=0) for k in keys) * np.sqrt((q ** 2).sum(2)).max()
    loose = EPSILON_32 * (64 + max(map(len, keys)) / 8 + 2 * (SIZE + 6) * score)
    near(got[0], out, (weight + loose) * sizes + far + ROUNDING[world.kind] * np.abs(out) + TINY[world.kind],
         "out")
    near(got[1], normalizers, loose + 4 * EPSILON_32 * np.abs(normalizers), "normalizers")


def far(world):
    """What weights below f16's numbers may be off by, times the values."""
    if world.kind != lib.F16 or world.fmt == lib.CACHE_INT8:
        return 0.0
    finite = lambda t: np.where(np.isfinite(t), t, 0.0)
    return 2.0**-31 * max(np.abs(finite(world.rows(1, h, s))).sum(0).max()
                          for h in range(world.key_heads) for s in range(len(world.lengths)))


# Of common and of uncommon values, 2^30 apart (f16, whose results have to be
# in its range, 2^22).
SPREAD = {lib.F32: (1.0, 2.0**30), lib.BF16: (1.0, 2.0**30), lib.F16: (2.0**-8, 2.0**14)}


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("lengths,new,prefix,heads", [([70, 40], [4, 3], 0, 2), ([33, 200], [3, 8], 50, 2),
                                                      ([90], [40], 0, 4), ([45, 60], [30, 30], 70, 4)])
def test_large_values_that_are_not_seen(kind, lengths, new, prefix, heads):
    # The last token's value in 8 bits, which those before it do not see.
    world = World(kind, lib.CACHE_INT8, 1, SIZE, 16, lengths, new, prefix)
    rng = np.random.default_rng(1)
    low, high = SPREAD[kind]
    world.fill(rng)
    world.scales[1] *= np.float32(low)
    for s, n in enumerate(lengths):
        world.put(world.slot(world.table[s], n - 1), 1, high * rng.standard_normal((1, SIZE)))
    world.upload()
    q = queries(world, heads)
    check(world, q, run(world, q, SCALE), 0.0 if kind == lib.F32 else 2.0**-16)


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("length,prefix", [(100, 0), (9, 200), (600, 0)])
def test_large_values_of_little_weight(kind, length, prefix):
    # Rows that a query sees with a score far below the others', so that they
    # add nothing, or about as much as these.
    world = World(kind, lib.CACHE_INT8, 2, SIZE, 16, [length], prefix=prefix)
    rng = np.random.default_rng(2)
    low, high = SPREAD[kind]
    world.fill(rng)
    world.scales[1] *= np.float32(low)
    q = queries(world, 2)
    pages, count = (world.prefix_pages, prefix) if prefix else (world.table[0], length)
    for at, score in ((5, -60.0), (count // 2, -np.log(high / low)), (count - 3, -90.0)):
        place = world.slot(pages, at)
        world.put(place, 0, score * q[0] / (SCALE * (q[0] ** 2).sum(1, keepdims=True)))
        world.put(place, 1, high * rng.standard_normal((2, SIZE)))
    world.upload()
    check(world, q, run(world, q, SCALE), 0.0 if kind == lib.F32 else 2.0**-16)


class Alike(World):
    """`count` sequences on the same pages, `new` tokens of each a call's: many
    tiles for a block, of few rows in the cache."""

    def __init__(self, kind, fmt, key_heads, size, page, length, count, new=1, seed=0):
        super().__init__(kind, fmt, key_heads, size, page, [length], [new], seed=seed)
        self.lengths, self.new = [length] * count, [new] * count
        self.table = np.repeat(self.table, count, 0)
        self.offsets = (new * np.arange(count + 1)).astype(np.uint32)
        self.tokens = new * count
        self.held = {}

    def fill(self, rng, spread=1.0):
        self.lengths, whole = self.lengths[:1], self.lengths
        super().fill(rng, spread)
        self.lengths = whole

    def rows(self, n, head, sequence):
        if (n, head) not in self.held:
            self.held[n, head] = super().rows(n, head, 0)
        return self.held[n, head]


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("fmt", [lib.CACHE_PLAIN, lib.CACHE_INT8])
@pytest.mark.parametrize("new,heads,count", [(1, 2, 40), (8, 8, 40)])
def test_infinities_and_nans_that_later_scores_outweigh(kind, fmt, new, heads, count):
    # Rows of 4 and of 64 queries, several tiles a wave.  A score 800 below the
    # largest has a weight of 0 in 64 bits too: what is infinite there is a NaN.
    world = Alike(kind, fmt, 2, SIZE, 16, 1024, count, new)
    rng = np.random.default_rng(3)
    world.fill(rng)
    one = queries(world, 2)[0]
    q = np.broadcast_to(np.repeat(one, heads // 2, 0), (world.tokens, heads, SIZE)).copy()
    for at in range(32, 300, 16):
        rows = 800.0 * one / (SCALE * (one ** 2).sum(1, keepdims=True))
        world.put(world.slot(world.table[0], at + 2), 0, rows + 0.01 * rng.standard_normal(rows.shape))
    for at, what in ((3, np.nan), (4, np.inf), (5, -np.inf)):
        rows = rng.standard_normal((2, SIZE))
        rows[:, 2 * at] = what
        world.put(world.slot(world.table[0], at), 1, rows)
    world.upload()
    got = run(world, q, SCALE)
    assert np.isnan(got[0][..., [6, 8, 10]]).all()
    if fmt == lib.CACHE_PLAIN:
        assert np.isfinite(got[0]).sum() == world.tokens * heads * (SIZE - 3)
        check(world, q, got, WEIGHT[kind], far(world))


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("fmt", [lib.CACHE_PLAIN, lib.CACHE_INT8])
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("lengths,new,prefix", [([90], [40], 0), ([45, 80], [30, 30], 70)])
def test_what_later_tokens_hold_where_many_rows_share_keys(kind, fmt, what, lengths, new, prefix):
    world = World(kind, fmt, 1, SIZE, 16, lengths, new, prefix)
    rng = np.random.default_rng(4)
    world.fill(rng)
    for s, (n, own) in enumerate(zip(lengths, new)):
        for pool, at, element in ((0, n - 1, 5), (1, n - 1, 6), (1, n - 9, 9), (1, n - own // 2, 11)):
            rows = rng.standard_normal((1, SIZE))
            rows[0, element] = what
            world.put(world.slot(world.table[s], at), pool, rows)
    world.upload()
    q = queries(world, 4)
    got = run(world, q, SCALE)
    first = np.cumsum([0] + new)
    for s, own in enumerate(new):
        mine = got[0][first[s]:first[s + 1]]
        assert np.isfinite(mine[:own // 2]).all() and not np.isfinite(mine[-9:]).all((1, 2)).any()
    attention_check(world, q, SCALE, got)


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("fmt", [lib.CACHE_PLAIN, lib.CACHE_INT8])
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("heads", [2, 8])
def test_what_a_prefix_holds(kind, fmt, what, heads):
    # 6 rows over the prefix, and 24.
    world = World(kind, fmt, 1, SIZE, 16, [20, 5, 40], prefix=150)
    rng = np.random.default_rng(5)
    world.fill(rng)
    for at, element in ((0, 3), (70, 7), (149, 7)):
        rows = rng.standard_normal((1, SIZE))
        rows[0, element] = what
        world.put(world.slot(world.prefix_pages, at), 1, rows)
    world.upload()
    q = queries(world, heads)
    got = run(world, q, SCALE)
    attention_check(world, q, SCALE, got)
    if fmt == lib.CACHE_PLAIN:
        assert not np.isfinite(got[0][..., [3, 7]]).any() and np.isfinite(np.delete(got[0], [3, 7], 2)).all()


@pytest.mark.parametrize("kind", [lib.F16, lib.BF16], ids=KIND_NAMES.get)
@pytest.mark.parametrize("fmt", [lib.CACHE_PLAIN, lib.CACHE_INT8])
@pytest.mark.parametrize("lengths,new,prefix,heads", [([700, 90, 333], None, 0, 24), ([300, 90], [20, 9], 200, 8)])
def test_weights_keep_their_bits(kind, fmt, lengths, new, prefix, heads):
    # The root of the mean square of all errors is that of the results' rounding
    # alone, half a step over the root of 3 each: weights of 2^-11 made it 1.14 to
    # 1.43 times that in f16.  (The mean square of 2000 has a deviation of 2%, and
    # what 32 bits add, 2^-24 of some 10 roundings, is below 1% of f16's.)
    world = World(kind, fmt, 2, SIZE, 16, lengths, new, prefix)
    world.fill(np.random.default_rng(6))
    world.upload()
    q = queries(world, heads)
    got, _ = run(world, q, SCALE)
    out, _, _ = generation.cache_attention(world, q, SCALE)
    half_step = ROUNDING[kind] * 2.0 ** np.floor(np.log2(np.abs(out)))
    assert ((got - out) ** 2).mean() ** 0.5 < 1.1 * (half_step ** 2 / 3).mean() ** 0.5


@pytest.mark.parametrize("prefix", [0, 90])
def test_a_prompt_without_pages_of_its_own(prefix):
    # It sees the prefix alone, and where there is none nothing.
    world = World(lib.BF16, lib.CACHE_PLAIN, 1, SIZE, 16, [0, 0], [700, 30], prefix, extra=0)
    world.fill(np.random.default_rng(7))
    world.lengths = [700, 30]
    world.upload()
    q = queries(world, 4)
    got = run(world, q, SCALE)
    attention_check(world, q, SCALE, got)
    assert prefix or ((got[0] == 0).all() and (got[1] == -np.inf).all())


@pytest.mark.parametrize("fmt", [lib.CACHE_PLAIN, lib.CACHE_INT8])
def test_keys_on_no_page_count_and_keys_behind_all_pages_do_not(fmt):
    # A sequence of 48 tokens on two pages of 16 and one that is none, and with a
    # table of the two alone.
    world = World(lib.F32, fmt, 1, SIZE, 16, [32], [1], extra=0)
    world.fill(np.random.default_rng(8))
    q = queries(world, 2)
    results, totals = [], []
    for most in (3, 2):
        world.table = np.concatenate([world.table[:, :2], np.full((1, most - 2), world.page_count, np.uint32)], 1)
        world.most, world.lengths = most, [48]
        world.upload()
        got, normalizers = run(world, q, SCALE)
        results.append(got[0])
        totals.append(np.exp(normalizers))
    # 16 keys of score 0 more, in f32: some 100 roundings of the sums.
    assert np.abs(totals[0] - totals[1] - 16).max() < 100 * EPSILON_32 * totals[0].max()
    sums = [r * t for r, t in zip(results, totals)]
    assert np.abs(sums[0] - sums[1]).max() < 100 * EPSILON_32 * 4 * totals[0].max()  # values to 4


@pytest.mark.parametrize("kind", [lib.F32, lib.BF16], ids=KIND_NAMES.get)
@pytest.mark.parametrize("fmt", [lib.CACHE_PLAIN, lib.CACHE_INT8])
@pytest.mark.parametrize("power", [-100, 100])
def test_values_near_the_ends_of_the_range(kind, fmt, power):
    # 100 keys of values to some 2^102, times the weights' 2^8: below 2^117.
    world = World(kind, fmt, 1, SIZE, 16, [100, 17], [2, 1])
    rng = np.random.default_rng(9)
    world.fill(rng)
    for s, n in enumerate(world.lengths):
        for at in range(n):
            world.put(world.slot(world.table[s], at), 1, rng.standard_normal((1, SIZE)) * 2.0**power)
    world.upload()
    q = queries(world, 2)
    check(world, q, run(world, q, SCALE), WEIGHT[kind])
