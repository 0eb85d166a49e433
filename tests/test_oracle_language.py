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
