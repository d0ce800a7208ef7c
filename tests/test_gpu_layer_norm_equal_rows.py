"""Rows of equal elements: the mean is that element, and the result the bias, to the bit.

Of N equal elements v the sums leave a first mean k steps of v's last place beside v
with k below 90, the differences from it and their sum, k N of those steps, are whole
numbers of them and exact, and so is the quotient: what is left of the row after both
parts of the mean is zero.  The sum of squares, k^2 N, is exact below 2^24 as well;
the variance is then zero and without epsilon 0 / 0 is left.
"""
import numpy as np
import pytest

from test_gpu_layer_norm import ctx, run_backward, run_forward  # noqa: F401 (ctx is a fixture)

pytestmark = pytest.mark.gpu

# lengths whose reciprocals are rounded the wrong way for some multiple, in every shape of the kernels
COLS = [41, 83, 107, 141, 249, 497, 511, 1284, 1621, 1810, 4099, 8193, 29761, 32768, 40001, 100003]


@pytest.mark.parametrize("t", [np.float32, np.float64])
@pytest.mark.parametrize("cols", COLS)
def test_the_result_is_the_bias(ctx, cols, t):
    rng = np.random.default_rng(cols)
    values = (rng.uniform(1, 2, 60) * 10.0 ** rng.integers(-3, 9, 60) * rng.choice([-1, 1], 60)).astype(t)
    x = np.repeat(values[:, None], cols, 1)
    w, b = rng.normal(1, 0.2, cols).astype(t), rng.normal(0, 1, cols).astype(t)
    for eps in (1e-5, 1e-12):
        y, mean, rstd = run_forward(ctx, x, w, b, eps, pad=1)
        np.testing.assert_array_equal(y, np.repeat(b[None], 60, 0))
        np.testing.assert_array_equal(mean, values)
        y, _, _ = run_forward(ctx, x, w, None, eps, stats=False)
        assert not y.any()
    g = rng.normal(0, 1, x.shape).astype(t)
    assert not run_backward(ctx, g, x, w, 1e-5, want=("dw",))["dw"].any()


@pytest.mark.parametrize("cols", [c for c in COLS if c < 3000])
def test_without_epsilon_nothing_is_left(ctx, cols):
    """(Up to 3000 elements k is below 70.)"""
    rng = np.random.default_rng(cols)
    values = (rng.uniform(1, 2, 60) * 10.0 ** rng.integers(-3, 9, 60)).astype(np.float32)
    y, _, _ = run_forward(ctx, np.repeat(values[:, None], cols, 1), None, None, 0.0)
    assert np.isnan(y).all()


@pytest.mark.parametrize("cols", [83, 511, 4099, 40001])
def test_deviations_that_cannot_be_squared(ctx, cols):
    """Beyond 2^63 in float the variance is infinite and the result the bias, as it was."""
    t = np.float32
    x = np.random.default_rng(cols).normal(0, 1e25, (3, cols)).astype(t)
    b = np.arange(cols, dtype=t)
    y, _, rstd = run_forward(ctx, x, None, b, 1e-5)
    if cols < 33000:
        np.testing.assert_array_equal(y, np.repeat(b[None], 3, 0))
        assert not rstd.any()


@pytest.mark.parametrize("t", [np.float32, np.float64])
@pytest.mark.parametrize("cols", [5, 83, 5000, 40001])
def test_the_smallest_epsilon_is_one(ctx, cols, t):
    """Below the type's numbers too: h is 0, and with it dweight."""
    rng = np.random.default_rng(cols)
    x = np.repeat(rng.uniform(1, 2, 4).astype(t)[:, None], cols, 1)
    b, g = rng.normal(0, 1, cols).astype(t), rng.normal(0, 1, x.shape).astype(t)
    for eps in (1e-50, 1e-310, 5e-324):
        y, _, rstd = run_forward(ctx, x, None, b, eps)
        np.testing.assert_array_equal(y, np.repeat(b[None], 4, 0))
        assert np.isfinite(rstd).all()
        assert not run_backward(ctx, g, x, None, eps, want=("dw",))["dw"].any()
