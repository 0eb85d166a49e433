"""What the operators of generation refuse, on the host and before any device
work (no test here touches a device)."""

import ctypes

from tensorcrate_amd import lib
from tests.test_language_refusals import refused


def test_the_rotary_shape_is_the_headers():
    # Natural C alignment of `tc_rotary_shape`.
    assert lib.RotaryShape.epsilon.offset == 32 and lib.RotaryShape.tokens.offset == 40
    assert lib.RotaryShape.frequencies.offset == 56 and ctypes.sizeof(lib.RotaryShape) == 64 + 8 * 8


def test_rotary_norm():
    def shape(dtype=lib.F32, weight=lib.F32, tokens=10, heads=4, key_heads=2, size=16, count=16, pairs=lib.HALVES,
              normalize=True, epsilon=1e-5, positions=64, frequencies=64, query=(64, 16), key=(32, 16),
              query_out=(64, 16), key_out=(32, 16)):
        return lib.rotary(dtype, weight, tokens, heads, key_heads, size, count, pairs, normalize, epsilon, positions,
                          frequencies, query, key, query_out, key_out)

    forward = lambda given, *operands: refused("tc_rotary_norm", given, *(operands or [64] * 6))
    back = lambda given, *operands: refused("tc_rotary_norm_backward", given, *(operands or [64] * 10))
    for run, what in ((forward, "rotary norm"), (back, "rotary norm, backward")):
        assert run(None) == (lib.INVALID, f"{what}: no shape")
        assert run(shape(dtype=lib.F64)) == (lib.UNSUPPORTED, f"{what}: no kernel for f64")
        assert run(shape(dtype=lib.F16, weight=lib.BF16)) == (
            lib.UNSUPPORTED, f"{what}: no kernel for f16 heads with a bf16 weight")
        assert run(shape(size=0, count=0)) == (lib.INVALID, f"{what}: heads of no elements")
        assert run(shape(size=129, query=(516, 129), key=(258, 129), query_out=(516, 129), key_out=(258, 129))) == (
            lib.UNSUPPORTED, f"{what}: heads of 129 elements, more than 128")
        for count in (3, 18):
            assert run(shape(count=count)) == (lib.INVALID, f"{what}: {count} rotated of 16 elements")
        assert run(shape(pairs=2)) == (lib.INVALID, f"{what}: pairs of kind 2")
        for epsilon in (-1.0, float("nan"), float("inf")):
            assert run(shape(epsilon=epsilon))[0] == lib.INVALID
        assert run(shape(normalize=False)) == (lib.INVALID, f"{what}: a weight without a norm")
        for name in ("query", "key", "query_out", "key_out"):
            for steps in ((16, 16), (64, 15), (0, 16), (16, 0), (2**62, 16), (16, 2**62)):
                assert run(shape(**{name: steps}))[0] == lib.INVALID, (name, steps)
        assert run(shape(tokens=2**32))[0] == lib.UNSUPPORTED
        assert run(shape(frequencies=None)) == (lib.INVALID, f"{what}: a null operand")
    for missing in (0, 1, 4, 5):
        operands = [64] * 6
        operands[missing] = None
        assert forward(shape(), *operands) == (lib.INVALID, "rotary norm: a null operand")
    for missing in (0, 1, 2, 3, 6, 7):
        operands = [64] * 10
        operands[missing] = None
        assert back(shape(), *operands) == (lib.INVALID, "rotary norm, backward: a null operand")
    # Weights' gradients belong to the norm too.
    assert back(shape(normalize=False), 64, 64, None, None, None, None, 64, 64, 64, None)[0] == lib.INVALID
    # Nothing to do, and no device needed.
    assert forward(shape(tokens=0), *[None] * 6)[0] == lib.OK
    assert back(shape(tokens=0), *[None] * 10)[0] == lib.OK


def test_the_cache_structs_are_the_headers():
    # Natural C alignment of `tc_cache` and `tc_cache_batch`.
    assert lib.Cache.keys.offset == 24 and ctypes.sizeof(lib.Cache) == 56
    assert lib.CacheBatch.offsets.offset == 24 and ctypes.sizeof(lib.CacheBatch) == 56


def pool(dtype=lib.F32, fmt=lib.CACHE_PLAIN, heads=2, size=16, page=8, pages=10, keys=64, values=64, key_scales=64,
         value_scales=64):
    return lib.cache(dtype, fmt, heads, size, page, pages, keys, values, key_scales, value_scales)


def batch(tokens=3, sequences=3, offsets=None, lengths=64, pages=64, most=4, prefix=0, prefix_pages=None):
    return lib.cache_batch(tokens, sequences, offsets, lengths, pages, most, prefix, prefix_pages)


def test_cache_bytes():
    for dtype, fmt, size, want in ((lib.F32, lib.CACHE_PLAIN, 16, 64), (lib.F32, lib.CACHE_PLAIN, 17, 80),
                                   (lib.BF16, lib.CACHE_PLAIN, 17, 48), (lib.F16, lib.CACHE_PLAIN, 128, 256),
                                   (lib.F32, lib.CACHE_INT8, 17, 32), (lib.BF16, lib.CACHE_INT8, 128, 128),
                                   (lib.F16, lib.CACHE_INT8, 1, 16)):
        entries, scales = lib.cache_bytes(pool(dtype, fmt, size=size))
        assert entries == 10 * 2 * 8 * want and scales == (10 * 2 * 8 * 4 if fmt == lib.CACHE_INT8 else 0)
    count = lib.u64()
    assert refused("tc_cache_bytes", pool(), None, ctypes.byref(count)) == (lib.INVALID, "cache: a null operand")
    assert refused("tc_cache_bytes", None, ctypes.byref(count), ctypes.byref(count))[0] == lib.INVALID
    # Many pages: counted in 64 bits.
    assert lib.cache_bytes(pool(lib.F32, size=128, heads=8, page=256, pages=2**20))[0] == 2**20 * 8 * 256 * 512


def test_the_cache_calls():
    step = (32, 16)
    write = lambda cache, batch, k=64, v=64, ks=step, vs=step: refused("tc_cache_write", cache, batch, k, *ks, v, *vs)
    read = lambda cache, batch, k=64, v=64, ks=step, vs=step: refused("tc_cache_read", cache, batch, k, *ks, v, *vs)
    attend = lambda cache, batch, q=64, o=64, ks=(64, 16), vs=(64, 16), heads=4, scale=0.25: refused(
        "tc_cache_attention", cache, batch, heads, scale, q, *ks, o, *vs, None)
    for run, what, names in ((write, "cache write", ("keys", "values")), (read, "cache read", ("keys", "values")),
                             (attend, "cache attention", ("queries", "results"))):
        invalid = lambda text: (lib.INVALID, f"{what}: {text}")
        assert run(None, batch()) == invalid("no cache")
        assert run(pool(), None) == invalid("no batch")
        assert run(pool(dtype=lib.F64), batch()) == (lib.UNSUPPORTED, f"{what}: no kernel for f64")
        assert run(pool(fmt=2), batch()) == invalid("a cache of format 2")
        assert run(pool(heads=0), batch()) == invalid("heads of no elements")
        assert run(pool(size=0), batch()) == invalid("heads of no elements")
        assert run(pool(size=129), batch()) == (lib.UNSUPPORTED, f"{what}: heads of 129 elements, more than 128")
        assert run(pool(page=0), batch()) == invalid("pages of no tokens")
        assert run(pool(pages=2**28), batch())[0] == lib.UNSUPPORTED
        assert run(pool(pages=2**32 - 1, heads=2**32 - 1, page=2**32 - 1), batch())[0] == lib.UNSUPPORTED
        assert run(pool(), batch(tokens=2**31))[0] == lib.UNSUPPORTED
        assert run(pool(), batch(sequences=2**24, offsets=64))[0] == lib.UNSUPPORTED
        assert run(pool(), batch(tokens=4)) == invalid("4 tokens of 3 sequences without offsets")
        assert run(pool(), batch(most=2**30))[0] == lib.UNSUPPORTED
        assert run(pool(), batch(lengths=None)) == invalid("a null operand")
        assert run(pool(), batch(pages=None)) == invalid("a null operand")
        assert run(pool(), batch(prefix=5)) == invalid("a null operand")
        assert run(pool(), batch(prefix=2**32 - 1, prefix_pages=64))[0] == lib.UNSUPPORTED
        for name in ("keys", "values"):
            assert run(pool(**{name: None}), batch()) == invalid("a null operand")
            assert run(pool(**{name: 72}), batch()) == invalid("keys or values that are not 16-byte aligned")
        for name in ("key_scales", "value_scales"):
            assert run(pool(fmt=lib.CACHE_INT8, **{name: None}), batch()) == invalid("a null operand")
        for given in (dict(k=None), dict(v=None)) if run is not attend else (dict(q=None), dict(o=None)):
            assert run(pool(), batch(), **given) == invalid("a null operand")
        for steps in ((16, 16), (64, 15), (0, 16), (16, 0), (2**62, 16), (16, 2**62)):
            for name, given in zip(names, ("ks", "vs")):
                status, text = run(pool(), batch(), **{given: steps})
                assert status == lib.INVALID and name in text, (steps, text)
        # No tokens: nothing is done, and no device is needed.
        assert run(pool(), batch(tokens=0, sequences=0), None, None)[0] == lib.OK
    for heads in (0, 1, 3):
        assert attend(pool(), batch(), heads=heads) == (
            lib.INVALID, f"cache attention: {heads} query heads do not share 2 key heads evenly")
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert attend(pool(), batch(), scale=scale)[0] == lib.INVALID
    assert attend(pool(), batch(tokens=2**29, sequences=1, offsets=64))[0] == lib.UNSUPPORTED
