"""The operators of generation together, as a program that answers token by
token uses them: queries and keys normed and rotated, keys and values written to
the cache, attention over it; and the same captured into a HIP graph."""

import threading

import numpy as np
import pytest

from tensorcrate_amd import lib
from tests import generation, language
from tests.common import KIND_NAMES, KINDS, CapturedGraph, to_kind
from tests.generation import NO_PAGE, Heads, World
from tests.language import EPSILON_32, ROUNDING, near, stored

pytestmark = pytest.mark.gpu

HEADS, KEY_HEADS, SIZE, PAGE = 6, 2, 40, 16


class Model:
    """One layer's projections of given tokens, for sequences over one cache."""

    def __init__(self, kind, fmt, lengths, seed=0):
        self.kind, self.fmt, self.lengths = kind, fmt, lengths
        rng = np.random.default_rng(seed)
        self.projections = [stored(rng.standard_normal((n, HEADS + 2 * KEY_HEADS, SIZE)), kind) for n in lengths]
        self.weights = [stored(1 + 0.2 * rng.standard_normal(SIZE), kind) for _ in range(2)]
        self.frequencies = (100.0 ** (-np.arange(SIZE // 2) / (SIZE // 2))).astype(np.float32)
        self.world = World(kind, fmt, KEY_HEADS, SIZE, PAGE, lengths)
        self.world.upload()
        self.device = [Heads(w.reshape(1, 1, SIZE), kind) for w in self.weights] + [lib.Buffer.of(self.frequencies)]
        self.scale = float(np.float32(SIZE ** -0.5))

    def step(self, begins, ends):
        """Tokens begins[s] to ends[s] of each sequence through the calls; their
        results."""
        kind, world = self.kind, self.world
        rows = np.concatenate([p[b:e] for p, b, e in zip(self.projections, begins, ends)])
        tokens = len(rows)
        projected = Heads(rows, kind)
        positions = lib.Buffer.of(np.concatenate([np.arange(b, e) for b, e in zip(begins, ends)]).astype(np.uint32))
        offsets = lib.Buffer.of(np.cumsum([0] + [e - b for b, e in zip(begins, ends)]).astype(np.uint32))
        lengths = lib.Buffer.of(np.array(ends, np.uint32))
        width = SIZE * lib.DTYPE_SIZE[kind]
        q, k, v = (projected.ptr + width * n for n in (0, HEADS, HEADS + KEY_HEADS))
        steps = projected.steps
        shape = lib.rotary(kind, kind, tokens, HEADS, KEY_HEADS, SIZE, SIZE, lib.HALVES, True, 1e-5, positions.ptr,
                           self.device[2].ptr, steps, steps, steps, steps)
        # In place, in the projection's output.
        lib.call("tc_rotary_norm", shape, q, k, self.device[0].ptr, self.device[1].ptr, q, k)
        batch = lib.cache_batch(tokens, len(self.lengths), offsets.ptr, lengths.ptr, world.tables[2].ptr, world.most)
        lib.call("tc_cache_write", world.cache, batch, k, *steps, v, *steps)
        out = Heads.empty(tokens, HEADS, SIZE, kind)
        lib.call("tc_cache_attention", world.cache, batch, HEADS, self.scale, q, *steps, out.ptr, *out.steps, None)
        got = out.read()
        return [got[b:e] for b, e in zip(np.cumsum([0] + [e - b for b, e in zip(begins, ends)]),
                                         np.cumsum([e - b for b, e in zip(begins, ends)]))]

    def exact(self):
        """All tokens' results in 64 bits, causal over their whole sequences."""
        results = []
        for rows in self.projections:
            positions = np.arange(len(rows))
            q, _ = generation.rotary(rows[:, :HEADS], self.weights[0], 1e-5, positions, self.frequencies, lib.HALVES)
            k, _ = generation.rotary(rows[:, HEADS:HEADS + KEY_HEADS], self.weights[1], 1e-5, positions, self.frequencies,
                                     lib.HALVES)
            results.append(language.attention(q, k, rows[:, HEADS + KEY_HEADS:], [0, len(rows)], self.scale)[0])
        return results


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("fmt", [lib.CACHE_PLAIN, lib.CACHE_INT8])
def test_prompts_then_tokens_give_the_whole_sequences_attention(kind, fmt):
    lengths = [70, 33, 50]
    model = Model(kind, fmt, lengths)
    prompts = [n - 9 for n in lengths]
    got = model.step([0] * 3, prompts)
    # Drafts of three tokens, then one by one.
    for count in (3, 1, 1, 1, 1, 1, 1):
        ends = [p + count for p in prompts]
        for g, new in zip(range(3), model.step(prompts, ends)):
            got[g] = np.concatenate([got[g], new])
        prompts = ends
    assert prompts == lengths
    # Keys and values are off by their rounding: to the type (queries too), in 8
    # bits by half a step of the row, |x| <= 4 sigma / 254 with rows of 40.  A
    # score moves by scale |q| |dk|, weights relatively by twice that at most,
    # results by that of |v| and by dv.
    for result, want, rows in zip(got, model.exact(), model.projections):
        v = np.abs(rows[:, HEADS + KEY_HEADS:]).max()
        row = np.sqrt(SIZE) * 1.8  # of a normed head, weights at most 1.8
        step = ROUNDING[kind] + (np.abs(rows).max() * 1.8 / 254 if fmt == lib.CACHE_INT8 else 0.0)
        moved = model.scale * (row * np.sqrt(SIZE) * step + row * row * ROUNDING[kind]) + 2.0**-16
        near(result, want, 2 * moved * v + 2 * step * v + 4 * ROUNDING[kind] * v, "results")


class Step:
    """A step's operands and results; `fill(seed)` makes new inputs in place,
    `run()` queues the calls and `read()` gives all results' bytes."""

    def __init__(self, kind, fmt, prefix):
        self.kind = kind
        self.world = World(kind, fmt, KEY_HEADS, SIZE, PAGE, [300, 5, 129, 64], [1, 2, 3, 1], prefix=prefix, trail=2)
        self.world.fill(np.random.default_rng(0))
        self.world.upload()
        self.tokens = self.world.tokens
        self.rows = Heads(np.zeros((self.tokens, HEADS + 2 * KEY_HEADS, SIZE)), kind)
        self.turned = Heads.empty(self.tokens, HEADS + 2 * KEY_HEADS, SIZE, kind)
        self.back = Heads.empty(self.tokens, HEADS + 2 * KEY_HEADS, SIZE, kind)
        self.out = Heads.empty(self.tokens, HEADS, SIZE, kind)
        self.kept = [Heads.empty(self.tokens, KEY_HEADS, SIZE, kind) for _ in range(2)]
        self.normalizers = lib.Buffer(4 * HEADS * self.tokens)
        self.weights = [Heads(np.ones((1, 1, SIZE)), kind) for _ in range(2)]
        self.dw = [Heads.empty(1, 1, SIZE, kind) for _ in range(2)]
        self.positions = lib.Buffer.of(np.arange(self.tokens, dtype=np.uint32) * 1000)
        self.frequencies = lib.Buffer.of(np.linspace(1, 0.001, SIZE // 2).astype(np.float32))
        steps = self.rows.steps
        self.shape = lib.rotary(kind, kind, self.tokens, HEADS, KEY_HEADS, SIZE, SIZE, lib.NEIGHBOURS, True, 1e-5,
                                self.positions.ptr, self.frequencies.ptr, steps, steps, steps, steps)

    def fill(self, seed):
        rng = np.random.default_rng(seed)
        values = to_kind(rng.standard_normal(self.rows.whole.size).astype(np.float32), self.kind)
        lib.call("tc_upload", self.rows.buffer.ptr, values.ctypes.data, values.nbytes)
        # Lengths change from step to step too; sequences grow and shrink.
        lengths = np.array([300 - 40 * seed, 5 + seed, 129 - seed, 64 - 20 * seed], np.uint32)
        lib.call("tc_upload", self.world.tables[1].ptr, lengths.ctypes.data, lengths.nbytes)

    def results(self):
        return [h.buffer for h in (self.turned, self.back, self.out, *self.kept, *self.dw)] + [self.normalizers]

    def spoil(self):
        for buffer in self.results():
            values = np.full(buffer.nbytes, 0x55, np.uint8)
            lib.call("tc_upload", buffer.ptr, values.ctypes.data, values.nbytes)

    def run(self):
        width = SIZE * lib.DTYPE_SIZE[self.kind]
        at = lambda h: [h.ptr + width * n for n in (0, HEADS, HEADS + KEY_HEADS)]
        w = [h.ptr for h in self.weights]
        lib.call("tc_rotary_norm", self.shape, *at(self.rows)[:2], *w, *at(self.turned)[:2])
        lib.call("tc_rotary_norm_backward", self.shape, *at(self.turned)[:2], *at(self.rows)[:2], *w, *at(self.back)[:2],
                 *(d.ptr for d in self.dw))
        k, v = at(self.turned)[1], at(self.rows)[2]
        lib.call("tc_cache_write", self.world.cache, self.world.batch, k, *self.turned.steps, v, *self.rows.steps)
        lib.call("tc_cache_attention", self.world.cache, self.world.batch, HEADS, 0.16, at(self.turned)[0],
                 *self.turned.steps, self.out.ptr, *self.out.steps, self.normalizers.ptr)
        lib.call("tc_cache_read", self.world.cache, self.world.batch, self.kept[0].ptr, *self.kept[0].steps,
                 self.kept[1].ptr, *self.kept[1].steps)

    def read(self):
        return [buffer.download(np.uint8).tobytes() for buffer in self.results()]


@pytest.mark.parametrize("kind", KINDS, ids=KIND_NAMES.get)
@pytest.mark.parametrize("fmt,prefix", [(lib.CACHE_PLAIN, 0), (lib.CACHE_INT8, 200), (lib.CACHE_PLAIN, 90)])
def test_replays_give_the_eager_results(kind, fmt, prefix):
    failures = []

    def captured():  # a thread, and with it a stream, of its own
        try:
            step = Step(kind, fmt, prefix)
            step.fill(1)
            step.run()
            lib.sync()
            graph = CapturedGraph(step.run)
            for seed in (1, 2, 0, 3, 2):
                step.fill(seed)
                step.spoil()
                step.run()
                want = step.read()
                step.spoil()
                graph.replay()
                got = step.read()
                failures.extend((seed, n) for n in range(len(want)) if got[n] != want[n])
            graph.close()
        except Exception as error:  # reported on the test's thread
            failures.append(repr(error))

    worker = threading.Thread(target=captured)
    worker.start()
    worker.join()
    assert not failures


def test_two_graphs_of_one_thread_do_not_share_their_parts():
    # Each graph's workspace is its own: replays in either order, one after the
    # other without waiting, give what each gives alone.
    failures = []

    def captured():
        try:
            steps = [Step(lib.BF16, lib.CACHE_INT8, 0), Step(lib.F32, lib.CACHE_PLAIN, 200)]
            for seed, step in enumerate(steps):
                step.fill(seed)
                step.spoil()  # what lies between the rows is compared too
                step.run()
            lib.sync()
            want = [step.read() for step in steps]
            graphs = [CapturedGraph(step.run) for step in steps]
            for order in ((0, 1), (1, 0), (0, 1, 0, 1)):
                for step in steps:
                    step.spoil()
                for n in order:
                    graphs[n].replay()
                failures.extend((order, n) for n in range(2) if steps[n].read() != want[n])
            for graph in graphs:
                graph.close()
        except Exception as error:
            failures.append(repr(error))

    worker = threading.Thread(target=captured)
    worker.start()
    worker.join()
    assert not failures
