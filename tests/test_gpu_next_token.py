"""The example that trains a small causal language model with layer norm,
attention, log probabilities and clipping together: its first gradients against
the same model in 64 bits, and that it learns."""

import numpy as np
import pytest

from examples.next_token import EPSILON, NONE, Model, sequences
from tests import language

pytestmark = pytest.mark.gpu


def gradients(p, inputs, targets, ends, heads, key_heads):
    """The model's mean log probability and gradients in 64 bits."""
    tokens, width = len(inputs), p["embedding"].shape[1]
    size, begin = width // heads, np.concatenate([[0], ends])
    norm = lambda n, x: language.layer_norm(x, p[f"norm {n} weight"], p[f"norm {n} bias"], EPSILON)
    rows = np.eye(p["embedding"].shape[0])[inputs]
    x1 = rows @ p["embedding"]
    a, m1, s1 = norm(1, x1)
    parts = np.split((a @ p["projection"]).reshape(tokens, -1, size), [heads, heads + key_heads], 1)
    out, normalizers, _ = language.attention(*parts, begin, size ** -0.5)
    mixed = out.reshape(tokens, -1)
    x2 = x1 + mixed @ p["attention out"]
    b, m2, s2 = norm(2, x2)
    z = b @ p["layer in"]
    h = np.maximum(z, 0)
    x3 = x2 + h @ p["layer out"]
    c, m3, s3 = norm(3, x3)
    logits = c @ p["logits"]
    chosen, totals, entropies, _, _ = language.log_probabilities(logits, targets, 0)
    counted = (targets < logits.shape[1]).sum()
    d = language.log_probabilities_backward(logits, targets, totals, entropies, np.full(tokens, -1.0 / counted),
                                            np.zeros(tokens))
    g = {"logits": c.T @ d}

    def norm_back(n, dy, x, m, s):
        dx, g[f"norm {n} weight"], g[f"norm {n} bias"] = language.layer_norm_backward(dy, x, p[f"norm {n} weight"], m, s)
        return dx

    dx = norm_back(3, d @ p["logits"].T, x3, m3, s3)
    g["layer out"] = h.T @ dx
    dz = (dx @ p["layer out"].T) * (z > 0)
    g["layer in"] = b.T @ dz
    dx = dx + norm_back(2, dz @ p["layer in"].T, x2, m2, s2)
    g["attention out"] = mixed.T @ dx
    back, _ = language.attention_backward((dx @ p["attention out"].T).reshape(out.shape), *parts, out, normalizers,
                                          begin, size ** -0.5)
    dq = np.concatenate(back, 1).reshape(tokens, -1)
    g["projection"] = a.T @ dq
    g["embedding"] = rows.T @ (dx + norm_back(1, dq @ p["projection"].T, x1, m1, s1))
    return chosen.sum() / counted, g


def test_first_gradients():
    model = Model(vocabulary=20, width=24, heads=4, key_heads=2, hidden=36, seed=3)
    inputs, targets, ends = sequences(np.random.default_rng(5), 20, 6)
    p = {name: np.squeeze(m.read().astype(np.float64), 0) if name.startswith("norm") else m.read().astype(np.float64)
         for name, m in model.parameters.items()}
    want, exact = gradients(p, inputs, targets, ends, 4, 2)
    got, grads = model.gradients(inputs, targets, ends)
    # Some twenty operations of f32 in a row, each off by a few 2^-24 of what
    # it adds up, over values of order 1.
    assert abs(got - want) < 1e-5
    for name, value in exact.items():
        have = grads[name].read().astype(np.float64).reshape(value.shape)
        assert np.abs(have - value).max() < 2e-5 * max(np.abs(value).max(), 1e-3) + 1e-7, name


def test_it_learns():
    model = Model(vocabulary=16, width=64, heads=4, key_heads=2, hidden=64)
    rng = np.random.default_rng(1)
    chosen, norms = zip(*(model.step(*sequences(rng, 16, 30)) for _ in range(200)))
    # Chance is log(1/16) = -2.8.  Knowing which tokens a sequence repeats, and
    # nothing of the present one, is a mean of log(1/2), log(1/3) and log(1/4):
    # -1.06.
    assert np.mean(chosen[:5]) < -2.0 and np.mean(chosen[-10:]) > -1.06
    assert all(np.isfinite(norms)) and max(norms) > 1.0  # so that some were clipped
