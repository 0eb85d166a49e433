"""Rows written into a cache of pages and read back, bit for bit."""

import numpy as np
import pytest

from tensorcrate_amd import lib
from tests.common import KINDS, to_kind, widen
from tests.generation import NO_PAGE, Heads, World
from tests.language import EPSILON_32, near, stored

pytestmark = pytest.mark.gpu

FORMATS = [lib.CACHE_PLAIN, lib.CACHE_INT8]


def operands(world, seed=0, layout={}, values=None):
    rng = np.random.default_rng(seed)
    shape = (world.tokens, world.key_heads, world.size)
    given = [stored(rng.standard_normal(shape) * np.exp(rng.standard_normal(shape[:2] + (1,))), world.kind)
             for _ in range(2)] if values is None else values
    return given, [Heads(g, world.kind, **layout) for g in given]


def write(world, held):
    k, v = held
    lib.call("tc_cache_write", world.cache, world.batch, k.ptr, *k.steps, v.ptr, *v.steps)


def read(world, layout={}):
    out = [Heads.empty(world.tokens, world.key_heads, world.size, world.kind, **layout) for _ in range(2)]
    lib.call("tc_cache_read", world.cache, world.batch, out[0].ptr, *out[0].steps, out[1].ptr, *out[1].steps)
    return [o.read() for o in out]


def check(world, layout={}, values=None, seed=0):
    """What is written is where it belongs, nothing else is, and it reads back."""
    world.upload()
    given, held = operands(world, seed, layout, values)
    write(world, held)
    want = [np.zeros((world.tokens, world.key_heads, world.size)) for _ in range(2)]
    for token, s, position in world.places():
        place = world.slot(world.table[s], position)
        for n in range(2):
            world.put(place, n, given[n][token])
            for head in range(world.key_heads):
                with np.errstate(over="ignore"):
                    want[n][token, head] = world.get(place, n, head).astype(np.float32)
    pools, scales = world.download()
    for n in range(2):
        assert pools[n].tobytes() == world.pools[n].tobytes(), "entries"
        # (A NaN's bits are not told.)
        assert np.array_equal(scales[n], world.scales[n], equal_nan=True), "scales"
    for got, expected in zip(read(world, layout), want):
        with np.errstate(over="ignore"):
            expected = widen(world.kind, to_kind(expected.astype(np.float32), world.kind))
        assert np.array_equal(got, expected, equal_nan=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("size,page,key_heads", [(1, 1, 1), (7, 3, 2), (16, 16, 8), (64, 5, 3), (75, 20, 3), (80, 48, 5),
                                                 (127, 7, 1), (128, 64, 9)])
def test_sizes(kind, fmt, size, page, key_heads):
    check(World(kind, fmt, key_heads, size, page, [1, 9, 30, 2 * page, 2 * page + 1]))
    check(World(kind, fmt, key_heads, size, page, [40, 1, 17], new=[40, 1, 5]), layout=dict(gap=3, token_gap=5, shift=1))


@pytest.mark.parametrize("fmt", FORMATS)
def test_sequences(fmt):
    for world in (World(lib.F16, fmt, 2, 24, 4, [5, 8, 3], new=[0, 3, 0], lead=2, trail=3),
                  World(lib.F16, fmt, 2, 24, 4, [5, 8, 3], new=[0, 0, 0], lead=4),
                  World(lib.F16, fmt, 2, 24, 4, [], new=[], lead=4),
                  # More tokens than the sequence has: those before it have no place.
                  World(lib.F16, fmt, 2, 24, 4, [5, 0, 3], new=[7, 2, 3]),
                  World(lib.F16, fmt, 3, 40, 4, list(range(1, 200)), new=[min(1 + n % 3, 1 + n) for n in range(199)], trail=1),
                  World(lib.F16, fmt, 1, 16, 16, [300] * 90, new=[260] + [1] * 89)):
        check(world)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("fmt", FORMATS)
def test_many_tokens(kind, fmt):
    check(World(kind, fmt, 9, 48, 100, [3000, 7], new=[2400, 7]))


@pytest.mark.parametrize("fmt", FORMATS)
def test_pages_that_are_none(fmt):
    world = World(lib.BF16, fmt, 2, 32, 4, [9, 12, 4], new=[9, 12, 4])
    world.table[0, 1] = world.page_count
    world.table[1, 2] = NO_PAGE
    world.lengths[2] = 7  # past its pages: the table's next one is none
    check(world)
    world = World(lib.BF16, fmt, 2, 32, 4, [9, 12], new=[9, 3], extra=0)
    world.lengths = [9, 14]  # past the table
    check(world)


@pytest.mark.parametrize("kind", KINDS)
def test_rows_that_are_hard_in_8_bits(kind):
    world = World(kind, lib.CACHE_INT8, 1, 20, 8, [12], new=[12])
    rng = np.random.default_rng(5)
    rows = rng.standard_normal((12, 1, 20))
    rows[0] = 0.0
    rows[1] = -0.0
    rows[2, 0, 3] = np.inf
    rows[3, 0, 0] = -np.inf
    rows[4, 0, 19] = np.nan
    rows[5] = {lib.F32: 1e-44, lib.F16: 2.0**-24, lib.BF16: 2.0**-133}[kind] * rng.integers(-3, 4, 20)
    rows[6] = {lib.F32: 3.4028235e38, lib.F16: 65504.0, lib.BF16: 3.3895314e38}[kind] * rng.choice([-1, 1, 0.5], 20)
    rows[7] = np.arange(20) * 0.5 * 127 / 64  # on and next to ties
    rows[8, 0, :] = 127.0 * np.sign(rows[8, 0, :])
    rows[9] = np.arange(-10, 10) + 0.5
    rows[9, 0, 0] = 127.0
    rows[10] = 1e-30
    rows[10, 0, 7] = 60000.0
    values = [stored(rows, kind), stored(rows[::-1], kind)]
    check(world, values=values)


def test_a_pool_of_no_pages():
    world = World(lib.F32, lib.CACHE_PLAIN, 2, 8, 4, [3])
    world.upload()
    world.cache.page_count = 0
    world.cache.keys = world.cache.values = None
    _, held = operands(world)
    write(world, held)
    assert all((r == 0).all() for r in read(world))


def test_rows_past_32_bits_of_bytes():
    # A pool of over 4 GiB, its last page past that, and the others untouched.
    pages, page, size = 4200, 256, 128
    cache = lib.cache(lib.F32, lib.CACHE_PLAIN, 8, size, page, pages, None, None)
    entries, _ = lib.cache_bytes(cache)
    assert entries > 2**32
    pools = [lib.Buffer(entries) for _ in range(2)]
    cache.keys, cache.values = (p.ptr for p in pools)
    table, lengths = lib.Buffer.of(np.array([pages - 1], np.uint32)), lib.Buffer.of(np.array([page], np.uint32))
    batch = lib.cache_batch(1, 1, None, lengths.ptr, table.ptr, 1)
    rows = np.random.default_rng(0).standard_normal((1, 8, size)).astype(np.float32)
    held = [Heads(rows, lib.F32), Heads(-rows, lib.F32)]
    lib.call("tc_cache_write", cache, batch, held[0].ptr, *held[0].steps, held[1].ptr, *held[1].steps)
    last = np.empty((8, page, size), np.float32)
    for n, sign in ((0, 1), (1, -1)):
        lib.call("tc_download", last.ctypes.data, pools[n].ptr + entries - last.nbytes, last.nbytes)
        assert np.array_equal(last[:, -1], sign * rows[0])
    q = Heads(rows, lib.F32)
    out = Heads.empty(1, 8, size, lib.F32)
    # A length of one puts the token at the page's first slot.
    lib.call("tc_upload", lengths.ptr, np.array([1], np.uint32).ctypes.data, 4)
    lib.call("tc_cache_write", cache, batch, held[0].ptr, *held[0].steps, held[1].ptr, *held[1].steps)
    lib.call("tc_cache_attention", cache, batch, 8, 0.1, q.ptr, *q.steps, out.ptr, *out.steps, None)
    # One key: (p v) (1 / p), three roundings of 32 bits.
    near(out.read(), -rows, 3.01 * EPSILON_32 * np.abs(rows), "one key")
