"""The language-model operators and their gradients captured into one HIP
graph: every replay, between eager calls and on inputs changed in place, gives
the eager calls' bits."""

import threading

import numpy as np
import pytest

from tensorcrate_amd import lib
from tests.common import CapturedGraph, to_kind

pytestmark = pytest.mark.gpu

F = lib.F32
TOKENS, WIDE, HEADS, KEY_HEADS, SIZE, VOCABULARY, ROWS = 300, 130, 6, 2, 40, 20001, 3
OFFSETS = np.array([2, 2, 71, 290], np.uint32)


class Step:
    """Operands and results of each operator; `fill(seed)` makes new inputs in
    place, `run()` queues the calls and `read()` gives all results' bytes."""

    def __init__(self, kind):
        self.kind, self.width = kind, lib.DTYPE_SIZE[kind]
        self.inputs, self.results = {}, {}
        for name, n in (("x", TOKENS * WIDE), ("dy", TOKENS * WIDE), ("w", WIDE), ("q", TOKENS * HEADS * SIZE),
                        ("k", TOKENS * KEY_HEADS * SIZE), ("v", TOKENS * KEY_HEADS * SIZE),
                        ("do", TOKENS * HEADS * SIZE), ("logits", ROWS * VOCABULARY)):
            self.inputs[name] = (lib.Buffer(n * self.width), n)
        for name, n in (("y", TOKENS * WIDE), ("dx", TOKENS * WIDE), ("dw", WIDE), ("db", WIDE),
                        ("o", TOKENS * HEADS * SIZE), ("dq", TOKENS * HEADS * SIZE),
                        ("dk", TOKENS * KEY_HEADS * SIZE), ("dv", TOKENS * KEY_HEADS * SIZE),
                        ("d_logits", ROWS * VOCABULARY), ("cx", TOKENS * WIDE), ("cw", WIDE)):
            self.results[name] = lib.Buffer(n * self.width)
        for name, n in (("means", TOKENS), ("scales", TOKENS), ("l", HEADS * TOKENS), ("lp", ROWS), ("z", ROWS),
                        ("h", ROWS), ("top", ROWS * 20), ("top tokens", ROWS * 20), ("norm", 1)):
            self.results[name] = lib.Buffer(n * 4)
        self.offsets = lib.Buffer.of(OFFSETS)
        self.tokens = lib.Buffer.of(np.array([5, VOCABULARY - 1, 0xFFFFFFFF], np.uint32))
        self.ones = lib.Buffer.of(np.ones(ROWS, np.float32))
        wide, narrow = (HEADS * SIZE, SIZE), (KEY_HEADS * SIZE, SIZE)
        self.shape = lib.attention(kind, TOKENS, HEADS, KEY_HEADS, SIZE, 0.2, self.offsets.ptr, len(OFFSETS) - 1, wide,
                                   narrow, narrow, wide)

    def fill(self, seed):
        rng = np.random.default_rng(seed)
        for buffer, n in self.inputs.values():
            values = to_kind(rng.standard_normal(n).astype(np.float32), self.kind)
            lib.call("tc_upload", buffer.ptr, values.ctypes.data, values.nbytes)

    def spoil(self):
        for buffer in self.results.values():
            values = np.full(buffer.nbytes, 0x55, np.uint8)
            lib.call("tc_upload", buffer.ptr, values.ctypes.data, values.nbytes)

    def run(self):
        i = {name: buffer.ptr for name, (buffer, _) in self.inputs.items()}
        r = {name: buffer.ptr for name, buffer in self.results.items()}
        kind = self.kind
        lib.call("tc_layer_norm", kind, kind, i["x"], WIDE, TOKENS, WIDE, i["w"], None, 1e-5, r["y"], WIDE, r["means"],
                 r["scales"])
        lib.call("tc_layer_norm_backward", kind, kind, i["dy"], WIDE, i["x"], WIDE, TOKENS, WIDE, i["w"], r["means"],
                 r["scales"], r["dx"], WIDE, r["dw"], r["db"])
        lib.call("tc_attention", lib.ctypes.byref(self.shape), i["q"], i["k"], i["v"], r["o"], r["l"])
        lib.call("tc_attention_backward", lib.ctypes.byref(self.shape), i["do"], i["q"], i["k"], i["v"], r["o"], r["l"],
                 r["dq"], r["dk"], r["dv"])
        lib.call("tc_log_probabilities", kind, i["logits"], VOCABULARY, ROWS, VOCABULARY, self.tokens.ptr, r["lp"],
                 r["z"], r["h"], 20, r["top"], r["top tokens"])
        lib.call("tc_log_probabilities_backward", kind, i["logits"], VOCABULARY, ROWS, VOCABULARY, self.tokens.ptr,
                 r["z"], r["h"], self.ones.ptr, self.ones.ptr, r["d_logits"], VOCABULARY)
        lib.call("tc_clip_global_norm", 2, (lib.u32 * 2)(kind, kind), (lib.vp * 2)(r["dx"], r["dw"]),
                 (lib.u64 * 2)(TOKENS * WIDE, WIDE), 1.0, (lib.vp * 2)(r["cx"], r["cw"]), r["norm"])

    def read(self):
        return {name: buffer.download(np.uint8).tobytes() for name, buffer in self.results.items()}


@pytest.mark.parametrize("kind", [lib.F32, lib.F16, lib.BF16])
def test_replays_give_the_eager_results(kind):
    failures = []

    def captured():  # a thread, and with it a stream, of its own
        try:
            step = Step(kind)
            step.fill(1)
            step.run()
            lib.sync()
            graph = CapturedGraph(step.run)
            for seed in (1, 2, 3, 2):
                step.fill(seed)
                step.spoil()
                step.run()
                want = step.read()
                step.spoil()
                graph.replay()
                got = step.read()
                failures.extend((seed, name) for name in want if got[name] != want[name])
            graph.close()
        except Exception as error:  # reported on the test's thread
            failures.append(repr(error))

    worker = threading.Thread(target=captured)
    worker.start()
    worker.join()
    assert not failures
