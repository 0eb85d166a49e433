"""What the language-model operators refuse, on the host and before any device
work (no test here touches a device)."""

import ctypes

from tensorcrate_amd import lib


def refused(name, *args):
    loaded = lib.load()
    status = getattr(loaded, name)(*args)
    return status, loaded.tc_last_error().decode()


def test_layer_norm():
    F, E = lib.F32, 1e-5
    assert refused("tc_layer_norm", lib.F64, F, 64, 8, 2, 8, None, None, E, 64, 8, None, None) == (
        lib.UNSUPPORTED, "layer norm: no kernel for f64")
    assert refused("tc_layer_norm", 9, F, 64, 8, 2, 8, None, None, E, 64, 8, None, None)[0] == lib.UNSUPPORTED
    assert refused("tc_layer_norm", lib.F16, lib.BF16, 64, 8, 2, 8, None, None, E, 64, 8, None, None) == (
        lib.UNSUPPORTED, "layer norm: no kernel for f16 rows with a bf16 weight")
    assert refused("tc_layer_norm", F, F, 64, 7, 2, 8, None, None, E, 64, 8, None, None) == (
        lib.INVALID, "layer norm: rows of 8 elements 7 apart overlap")
    assert refused("tc_layer_norm", F, F, 64, 8, 2, 8, None, None, E, 64, 5, None, None)[0] == lib.INVALID
    assert refused("tc_layer_norm", F, F, 64, 0, 2, 0, None, None, E, 64, 0, None, None) == (
        lib.INVALID, "layer norm: rows of no elements")
    assert refused("tc_layer_norm", F, F, 64, 2**25, 1, 2**25, None, None, E, 64, 2**25, None, None)[0] == lib.UNSUPPORTED
    assert refused("tc_layer_norm", F, F, None, 8, 2, 8, None, None, E, 64, 8, None, None) == (
        lib.INVALID, "layer norm: a null operand")
    assert refused("tc_layer_norm", F, F, 64, 8, 2, 8, None, None, E, None, 8, None, None)[0] == lib.INVALID
    assert refused("tc_layer_norm", F, F, 64, 2**40, 2**40, 2**30, None, None, E, 64, 2**40, None, None)[0] == lib.INVALID
    back = "tc_layer_norm_backward"
    assert refused(back, F, F, 64, 8, 64, 8, 2, 8, None, None, 64, 64, 8, None, None) == (
        lib.INVALID, "layer norm, backward: a null operand")
    assert refused(back, F, F, 64, 8, 64, 4, 2, 8, None, 64, 64, 64, 8, None, None)[0] == lib.INVALID
    assert refused(back, F, F, 64, 8, 64, 8, 2, 8, None, 64, 64, 64, 7, None, None)[0] == lib.INVALID
    assert refused(back, F, F, 64, 0, 64, 0, 2, 0, None, 64, 64, 64, 0, None, None) == (
        lib.INVALID, "layer norm, backward: rows of no elements")
    # Nothing wanted, or nothing there: nothing is done, and no device is needed.
    assert refused(back, F, F, 64, 8, 64, 8, 2, 8, None, 64, 64, None, 8, None, None)[0] == lib.OK


def test_log_probabilities():
    F = lib.F32
    run, back = "tc_log_probabilities", "tc_log_probabilities_backward"
    assert refused(run, lib.F64, 64, 8, 2, 8, None, None, 64, None, 0, None, None) == (
        lib.UNSUPPORTED, "log probabilities: no kernel for f64")
    assert refused(run, F, 64, 7, 2, 8, None, None, 64, None, 0, None, None) == (
        lib.INVALID, "log probabilities: rows of 8 elements 7 apart overlap")
    assert refused(run, F, 64, 800, 2, 800, None, None, 64, None, 65, 64, 64) == (
        lib.UNSUPPORTED, "log probabilities: the top 65 of at most 64")
    assert refused(run, F, 64, 8, 2, 8, None, None, 64, None, 9, 64, 64) == (
        lib.INVALID, "log probabilities: the top 9 of 8 logits")
    assert refused(run, F, 64, 0, 2, 0, None, None, 64, None, 0, None, None) == (
        lib.INVALID, "log probabilities: rows of no logits")
    null = (lib.INVALID, "log probabilities: a null operand")
    assert refused(run, F, None, 8, 2, 8, None, None, 64, None, 0, None, None) == null
    assert refused(run, F, 64, 8, 2, 8, 64, None, 64, None, 0, None, None) == null
    assert refused(run, F, 64, 8, 2, 8, None, 64, 64, None, 0, None, None) == null
    assert refused(run, F, 64, 8, 2, 8, None, None, 64, None, 2, 64, None) == null
    assert refused(run, F, 64, 2**33, 1, 2**32, None, None, 64, None, 0, None, None)[0] == lib.UNSUPPORTED
    null = (lib.INVALID, "log probabilities, backward: a null operand")
    assert refused(back, F, 64, 8, 2, 8, 64, None, None, 64, None, 64, 8) == null
    assert refused(back, F, 64, 8, 2, 8, None, 64, None, 64, None, 64, 8) == null
    assert refused(back, F, 64, 8, 2, 8, 64, 64, None, 64, 64, 64, 8) == null
    assert refused(back, F, 64, 8, 2, 8, 64, 64, 64, 64, 64, 64, 5)[0] == lib.INVALID


def test_clip():
    def arrays(*tensors):
        n = max(len(tensors), 1)
        kinds, pointers, lens = zip(*tensors)
        return (lib.u32 * n)(*kinds), (lib.vp * n)(*pointers), (lib.u64 * n)(*lens)

    kinds, tensors, lens = arrays((lib.F32, 64, 10), (lib.BF16, 64, 10))
    run = "tc_clip_global_norm"
    null = (lib.INVALID, "clip by global norm: a null operand")
    assert refused(run, 2, kinds, tensors, lens, -1.0, tensors, 64) == (
        lib.INVALID, "clip by global norm: a largest norm of -1.000000")
    assert refused(run, 2, kinds, tensors, lens, float("nan"), tensors, 64)[0] == lib.INVALID
    assert refused(run, 2, kinds, tensors, lens, 1.0, None, 64) == null
    assert refused(run, 2, kinds, tensors, lens, 1.0, tensors, None) == null
    assert refused(run, 2, None, tensors, lens, 1.0, tensors, 64) == null
    assert refused(run, 2, kinds, None, lens, 1.0, tensors, 64) == null
    assert refused(run, 2, kinds, tensors, None, 1.0, tensors, 64) == null
    assert refused(run, 2, kinds, tensors, lens, 1.0, arrays((0, 64, 0), (0, None, 0))[1], 64) == null
    some = arrays((lib.F32, 64, 10), (lib.BF16, None, 10))
    assert refused(run, 2, *some, 1.0, tensors, 64) == null
    assert refused("tc_global_norm", 2, *some, 64) == (lib.INVALID, "global norm: a null operand")
    some = arrays((lib.F32, 64, 10), (lib.F64, 64, 10))
    assert refused(run, 2, *some, 1.0, tensors, 64) == (lib.UNSUPPORTED, "clip by global norm: no kernel for f64")
    some = arrays((lib.F32, 64, 10), (lib.F32, 64, 2**41))
    assert refused("tc_global_norm", 2, *some, 64)[0] == lib.INVALID


def test_the_attention_shape_is_the_headers():
    # Natural C alignment of `tc_attention_shape`.
    assert ctypes.sizeof(lib.AttentionShape) == 4 * 4 + 8 + 4 + 4 + 8 + 8 * 8
    assert lib.AttentionShape.tokens.offset == 16 and lib.AttentionShape.offsets.offset == 32


def test_attention():
    def shape(dtype=lib.F32, tokens=10, heads=4, key_heads=2, size=16, scale=0.25, offsets=None, sequences=0,
              query=(64, 16), key=(32, 16), value=(32, 16), out=(64, 16)):
        return lib.attention(dtype, tokens, heads, key_heads, size, scale, offsets, sequences, query, key, value, out)

    def forward(given, *operands):
        return refused("tc_attention", given, *(operands or [64] * 5))

    back = lambda given, *operands: refused("tc_attention_backward", given, *(operands or [64] * 9))
    assert forward(None) == (lib.INVALID, "attention: no shape")
    assert forward(shape(dtype=lib.F64)) == (lib.UNSUPPORTED, "attention: no kernel for f64")
    for heads, key_heads in ((4, 3), (2, 4), (0, 1), (1, 0)):
        assert forward(shape(heads=heads, key_heads=key_heads)) == (
            lib.INVALID, f"attention: {heads} query heads do not share {key_heads} key heads evenly")
    assert forward(shape(size=0))[0] == lib.INVALID
    assert forward(shape(size=129, query=(516, 129), key=(258, 129), value=(258, 129), out=(516, 129))) == (
        lib.UNSUPPORTED, "attention: heads of 129 elements, more than 128")
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert forward(shape(scale=scale))[0] == lib.INVALID
    for name in ("query", "key", "value", "out"):
        for steps in ((16, 16), (64, 15), (0, 16), (16, 0), (2**62, 16), (16, 2**62)):
            assert forward(shape(**{name: steps}))[0] == lib.INVALID, (name, steps)
            assert back(shape(**{name: steps}))[0] == lib.INVALID, (name, steps)
    assert forward(shape(tokens=2**31))[0] == lib.UNSUPPORTED
    # 2^24 blocks and more are no dispatch: of tokens, of heads, of sequences.
    many = dict(heads=2**24, key_heads=2**24, size=1, query=(2**24, 1), key=(2**24, 1), value=(2**24, 1), out=(2**24, 1))
    assert forward(shape(tokens=1, **many))[0] == lib.UNSUPPORTED
    assert forward(shape(tokens=2**30, heads=4, key_heads=2))[0] == lib.UNSUPPORTED
    null = (lib.INVALID, "attention: a null operand")
    assert forward(shape(sequences=2)) == null
    for missing in range(4):
        operands = [64] * 5
        operands[missing] = None
        assert forward(shape(), *operands) == null
    for missing in range(9):
        operands = [64] * 9
        operands[missing] = None
        assert back(shape(), *operands) == (lib.INVALID, "attention, backward: a null operand")
