"""The plain gradients the language-model operators are checked against, held
to central differences of the plain forward passes in 64 bits."""

import numpy as np

from tests import language


def differences(f, x, step=1e-5):
    """The gradient of the scalar f at x, each from f at x +- step: off by
    f''' step^2 / 6 and by the rounding of f over step."""
    out = np.empty_like(x)
    for at in np.ndindex(x.shape):
        kept = x[at]
        x[at] = kept + step
        high = f()
        x[at] = kept - step
        low = f()
        x[at] = kept
        out[at] = (high - low) / (2 * step)
    return out


def test_layer_norm_gradients_are_the_differences():
    rng = np.random.default_rng(1)
    x, weight, bias = rng.standard_normal((3, 5)) * 2 + 1, rng.uniform(0.5, 1.5, 5), rng.standard_normal(5)
    dy = rng.standard_normal((3, 5))
    _, mean, scale = language.layer_norm(x, weight, bias, 1e-2)
    dx, dw, db = language.layer_norm_backward(dy, x, weight, mean, scale)
    loss = lambda: float((language.layer_norm(x, weight, bias, 1e-2)[0] * dy).sum())
    # Third derivatives of order 10 at these values: 1e-9 from the step, 1e-10 from rounding.
    assert np.allclose(dx, differences(loss, x), atol=1e-7)
    assert np.allclose(dw, differences(loss, weight), atol=1e-7)
    assert np.allclose(db, differences(loss, bias), atol=1e-7)


def test_log_probability_gradients_are_the_differences():
    rng = np.random.default_rng(2)
    x = rng.standard_normal((4, 6)) * 2
    tokens, d_given, d_entropies = np.array([1, 5, 6, 0]), rng.standard_normal(4), rng.standard_normal(4)
    given, normalizers, entropies, _, _ = language.log_probabilities(x, tokens, 0)
    d = language.log_probabilities_backward(x, tokens, normalizers, entropies, d_given, d_entropies)

    def loss():
        given, _, entropies, _, _ = language.log_probabilities(x, tokens, 0)
        return float((given * d_given).sum() + (entropies * d_entropies).sum())

    # Third derivatives below 10 here: 2e-10 from the step, 1e-10 from rounding.
    assert np.allclose(d, differences(loss, x), atol=1e-8)


def test_log_probabilities_of_impossible_tokens():
    x = np.array([[0.0, -np.inf, np.log(3.0)], [-np.inf] * 3])
    given, normalizers, entropies, top, tokens = language.log_probabilities(x, np.array([1, 0]), 3)
    assert np.array_equal(given, [-np.inf, -np.inf]) and np.allclose(normalizers[0], np.log(4.0))
    assert np.allclose(entropies, [np.log(4.0) - 0.75 * np.log(3.0), 0.0]) and normalizers[1] == -np.inf
    assert np.array_equal(tokens, [[2, 0, 1], [0, 1, 2]]) and np.allclose(top[0, :2], np.log([0.75, 0.25]))


def test_attention_gradients_are_the_differences():
    rng = np.random.default_rng(3)
    q, k, v, d = (rng.standard_normal((7, h, 3)) for h in (4, 2, 2, 4))
    ends, scale = [1, 1, 4, 6], 0.7
    out, normalizers, _ = language.attention(q, k, v, ends, scale)
    grads, _ = language.attention_backward(d, q, k, v, out, normalizers, ends, scale)
    loss = lambda: float((language.attention(q, k, v, ends, scale)[0] * d).sum())
    # Third derivatives below 10 here: 2e-10 from the step, 1e-10 from rounding.
    for name, grad, operand in zip("qkv", grads, (q, k, v)):
        assert np.allclose(grad, differences(loss, operand), atol=1e-8), name
    # What no sequence has, and the first token of each, whose softmax is of one.
    assert not out[[0, 6]].any() and not grads[0][[0, 1, 4, 6]].any()
    assert np.array_equal(out[1], np.repeat(v[1], 2, 0)) and np.isneginf(normalizers[:, [0, 6]]).all()
