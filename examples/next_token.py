"""A small causal language model trained on this backend: one block of
attention and a rectified layer between an embedding and a projection, each
behind a layer norm, on packed sequences of different lengths.

Every step runs the operators together as a training step uses them: layer
norm, attention over the packed sequences and the log probability of the next
token forward, their gradients backward, and the gradients clipped by their
common norm before Adam.  What lies between them are the products, sums and
updates that the backend has.

    python examples/next_token.py [steps]
"""

from __future__ import annotations

import sys
from pathlib import Path

import numpy as np

if str(Path(__file__).resolve().parent.parent) not in sys.path:
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from tensorcrate_amd import lib
from tensorcrate_amd.optim import Adam

F32 = lib.F32
EPSILON = 1e-5
NONE = 0xFFFFFFFF  # as a token: none


class Matrix:
    """rows x cols f32 on the device."""

    def __init__(self, rows: int, cols: int, values=None):
        self.rows, self.cols = rows, cols
        self.buffer = lib.Buffer(4 * rows * cols) if values is None else lib.Buffer.of(
            np.asarray(values, np.float32).reshape(rows, cols))

    @property
    def ptr(self) -> int:
        return self.buffer.ptr

    @property
    def size(self) -> int:
        return self.rows * self.cols

    def read(self) -> np.ndarray:
        return self.buffer.download(np.float32, self.size).reshape(self.rows, self.cols)


def product(form: int, a: Matrix, b: Matrix) -> Matrix:
    """a . b, or with LEFT a^T . b, or with RIGHT a . b^T."""
    m, k = (a.cols, a.rows) if form == lib.LEFT else (a.rows, a.cols)
    out = Matrix(m, b.rows if form == lib.RIGHT else b.cols)
    lib.call("tc_matmul", F32, F32, form, 0, m, k, out.cols, a.ptr, b.ptr, out.ptr)
    return out


def add(a: Matrix, b: Matrix) -> Matrix:
    out = Matrix(a.rows, a.cols)
    lib.call("tc_elementwise", F32, lib.ADD, a.ptr, b.ptr, out.ptr, a.size)
    return out


class Model:
    """Parameters by name, and a training step of them."""

    def __init__(self, vocabulary: int, width: int, heads: int, key_heads: int, hidden: int, rate: float = 3e-3,
                 limit: float = 1.0, seed: int = 0):
        rng = np.random.default_rng(seed)
        self.vocabulary, self.heads, self.key_heads, self.limit = vocabulary, heads, key_heads, limit
        self.head_size = width // heads
        columns = (heads + 2 * key_heads) * self.head_size
        normal = lambda rows, cols: Matrix(rows, cols, rng.standard_normal((rows, cols)) * rows ** -0.5)
        ones, zeros = (lambda: Matrix(1, width, np.ones(width))), (lambda: Matrix(1, width, np.zeros(width)))
        self.parameters = {
            "embedding": Matrix(vocabulary, width, rng.standard_normal((vocabulary, width)) * 0.5),
            "norm 1 weight": ones(), "norm 1 bias": zeros(), "projection": normal(width, columns),
            "attention out": normal(heads * self.head_size, width),
            "norm 2 weight": ones(), "norm 2 bias": zeros(), "layer in": normal(width, hidden),
            "layer out": normal(hidden, width),
            "norm 3 weight": ones(), "norm 3 bias": zeros(), "logits": normal(width, vocabulary),
        }
        self.rules = {name: Adam(rate) for name in self.parameters}

    def _norm(self, n: int, x: Matrix):
        y, means, scales = Matrix(x.rows, x.cols), Matrix(1, x.rows), Matrix(1, x.rows)
        weight, bias = (self.parameters[f"norm {n} {part}"] for part in ("weight", "bias"))
        lib.call("tc_layer_norm", F32, F32, x.ptr, x.cols, x.rows, x.cols, weight.ptr, bias.ptr, EPSILON, y.ptr,
                 y.cols, means.ptr, scales.ptr)

        def back(dy: Matrix, grads: dict) -> Matrix:
            dx = Matrix(x.rows, x.cols)
            dw, db = (grads.setdefault(f"norm {n} {part}", Matrix(1, x.cols)) for part in ("weight", "bias"))
            lib.call("tc_layer_norm_backward", F32, F32, dy.ptr, dy.cols, x.ptr, x.cols, x.rows, x.cols, weight.ptr,
                     means.ptr, scales.ptr, dx.ptr, dx.cols, dw.ptr, db.ptr)
            return dx

        return y, back

    def _attention(self, projected: Matrix, offsets: lib.Buffer, sequences: int):
        """Queries, keys and values side by side in a row of `projected`."""
        tokens, size = projected.rows, self.head_size
        out, normalizers = Matrix(tokens, self.heads * size), Matrix(self.heads, tokens)
        at = lambda m: [m.ptr + 4 * size * first for first in (0, self.heads, self.heads + self.key_heads)]
        packed = (projected.cols, size)
        shape = lib.attention(F32, tokens, self.heads, self.key_heads, size, size ** -0.5, offsets.ptr, sequences,
                              packed, packed, packed, (out.cols, size))
        lib.call("tc_attention", shape, *at(projected), out.ptr, normalizers.ptr)

        def back(d_out: Matrix) -> Matrix:
            d = Matrix(tokens, projected.cols)
            lib.call("tc_attention_backward", shape, d_out.ptr, *at(projected), out.ptr, normalizers.ptr, *at(d))
            return d

        return out, back

    def gradients(self, inputs: np.ndarray, targets: np.ndarray, ends):
        """(mean log probability of the targets, gradients by name) for tokens
        of sequences that end at `ends`; a target of NONE is not counted."""
        p, tokens = self.parameters, len(inputs)
        rows = Matrix(tokens, self.vocabulary, np.eye(self.vocabulary, dtype=np.float32)[inputs])
        offsets = lib.Buffer.of(np.concatenate([[0], ends]).astype(np.uint32))
        x = product(lib.PLAIN, rows, p["embedding"])
        a, norm_1_back = self._norm(1, x)
        mixed, attention_back = self._attention(product(lib.PLAIN, a, p["projection"]), offsets, len(ends))
        x = add(x, product(lib.PLAIN, mixed, p["attention out"]))
        b, norm_2_back = self._norm(2, x)
        z = product(lib.PLAIN, b, p["layer in"])
        h = Matrix(z.rows, z.cols)
        lib.call("tc_compare_scalar", F32, lib.MAX, z.ptr, 0.0, 0, h.ptr, z.size)
        x = add(x, product(lib.PLAIN, h, p["layer out"]))
        c, norm_3_back = self._norm(3, x)
        logits = product(lib.PLAIN, c, p["logits"])

        held = lib.Buffer.of(targets.astype(np.uint32))
        chosen, normalizers = Matrix(1, tokens), Matrix(1, tokens)
        lib.call("tc_log_probabilities", F32, logits.ptr, logits.cols, tokens, logits.cols, held.ptr, chosen.ptr,
                 normalizers.ptr, None, 0, None, None)
        counted = int((targets < self.vocabulary).sum())
        # The loss is the mean of -log p; its gradient takes the logits' place.
        d_chosen = Matrix(1, tokens, np.full(tokens, -1.0 / counted))
        lib.call("tc_log_probabilities_backward", F32, logits.ptr, logits.cols, tokens, logits.cols, held.ptr,
                 normalizers.ptr, None, d_chosen.ptr, None, logits.ptr, logits.cols)

        grads: dict[str, Matrix] = {"logits": product(lib.LEFT, c, logits)}
        dx = norm_3_back(product(lib.RIGHT, logits, p["logits"]), grads)
        grads["layer out"] = product(lib.LEFT, h, dx)
        dz, seen = product(lib.RIGHT, dx, p["layer out"]), Matrix(z.rows, z.cols)
        lib.call("tc_compare_scalar", F32, lib.GREATER, z.ptr, 0.0, 0, seen.ptr, z.size)
        lib.call("tc_elementwise", F32, lib.MUL, dz.ptr, seen.ptr, dz.ptr, z.size)
        grads["layer in"] = product(lib.LEFT, b, dz)
        dx = add(dx, norm_2_back(product(lib.RIGHT, dz, p["layer in"]), grads))
        grads["attention out"] = product(lib.LEFT, mixed, dx)
        d = attention_back(product(lib.RIGHT, dx, p["attention out"]))
        grads["projection"] = product(lib.LEFT, a, d)
        dx = add(dx, norm_1_back(product(lib.RIGHT, d, p["projection"]), grads))
        grads["embedding"] = product(lib.LEFT, rows, dx)
        return float(chosen.read().sum(dtype=np.float64) / counted), grads

    def step(self, inputs: np.ndarray, targets: np.ndarray, ends) -> tuple[float, float]:
        """One update; (mean log probability, norm of the gradients) before it."""
        chosen, grads = self.gradients(inputs, targets, ends)
        names = list(self.parameters)
        n, norm = len(names), Matrix(1, 1)
        at = (lib.vp * n)(*[grads[name].ptr for name in names])
        lib.call("tc_clip_global_norm", n, (lib.u32 * n)(*[F32] * n), at,
                 (lib.u64 * n)(*[grads[name].size for name in names]), self.limit, at, norm.ptr)
        for name in names:
            parameter = self.parameters[name]
            self.rules[name].update(parameter.buffer, grads[name].buffer, parameter.rows, parameter.cols)
        return chosen, float(norm.read()[0, 0])


def sequences(rng: np.random.Generator, vocabulary: int, count: int):
    """Packed sequences that repeat a short random pattern: what comes next can
    only be told by looking back.  (inputs, targets, ends)."""
    inputs, targets, ends = [], [], []
    for _ in range(count):
        length, period = int(rng.integers(8, 40)), int(rng.integers(2, 5))
        tokens = np.resize(rng.integers(0, vocabulary, period), length)
        inputs.append(tokens)
        targets.append(np.concatenate([tokens[1:], [NONE]]))
        # The first period is chance, and not asked for.
        targets[-1][:period - 1] = NONE
        ends.append(length)
    return np.concatenate(inputs), np.concatenate(targets), np.cumsum(ends)


def main(steps: int = 300) -> None:
    model = Model(vocabulary=32, width=64, heads=4, key_heads=2, hidden=128)
    rng = np.random.default_rng(1)
    for step in range(steps):
        chosen, norm = model.step(*sequences(rng, 32, 40))
        if step % 50 == 0 or step == steps - 1:
            print(f"step {step}: mean log probability {chosen:.3f}, gradient norm {norm:.3f}", flush=True)


if __name__ == "__main__":
    main(*map(int, sys.argv[1:2]))
