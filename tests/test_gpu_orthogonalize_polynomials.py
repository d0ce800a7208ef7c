"""tcg_orthogonalize with polynomials other than the usual one: which are taken and
which refused, and what those come to whose terms lie far apart.

Tolerances: as derived in test_gpu_orthogonalize, tol = eta sum_k D^(steps - 1 - k) |X_k|,
where eta allows for a B of norm 4 and an a of 4 at most.  A step rounds a X + B X, a
value of up to (|a| + F_k) |X_k| with F_k the largest norm of B, once and B by 2^-22 of
its norm: where a or F_k is larger, |X_k| counts max(1, F_k / 4, |a| / 4) times.
"""
import numpy as np
import pytest

from test_gpu_orthogonalize import ctx, eta, gradient, run  # noqa: F401 (ctx is a fixture)

pytestmark = pytest.mark.gpu


def close(got, g, steps, coef):
    a, b, c = coef
    x = g.astype(np.float64)
    x = x / (np.linalg.norm(x) + 1e-7)
    top, slopes, sizes = 1.0, [], []
    for _ in range(steps):
        s = np.linspace(0, top, 4001)
        slopes.append(max(abs(a + 3 * b * s ** 2 + 5 * c * s ** 4).max(), abs(a + b * s ** 2 + c * s ** 4).max(), 1.0))
        sizes.append(np.linalg.norm(x) * max(1.0, abs(b * s ** 2 + c * s ** 4).max() / 4, abs(a) / 4))
        top = abs(s * (a + b * s ** 2 + c * s ** 4)).max() * 1.001
        gram = x @ x.T
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    assert np.isfinite(got).all()
    tol = eta(g.dtype.type, g.shape) * sum(np.prod(slopes[k + 1:]) * sizes[k] for k in range(steps))
    off = np.linalg.norm(got.astype(np.float64) - x)
    assert off <= tol, "%g of the tolerance, %g of the result" % (off / tol, off / np.linalg.norm(x))


@pytest.mark.parametrize("rows,cols", [(40, 56), (300, 200)])
@pytest.mark.parametrize("t", [np.float32, np.float64])
@pytest.mark.parametrize("a,b", [(2.598, -2.598), (1.5, -0.5)])
def test_a_last_coefficient_that_is_almost_zero(ctx, rows, cols, t, a, b):
    """0.1 + 0.2 - 0.3 in place of nothing: the polynomial is largest where it is without that
    coefficient.  The term itself is below a rounding of every result."""
    g = gradient(rows, cols, t, seed=21)
    for c in (5.6e-17, 1e-18, -1e-17, 1e-300):
        close(run(ctx, g, steps=3, coef=(a, b, c))[0], g[0], 3, (a, b, 0.0))


@pytest.mark.parametrize("c", [0.0, 1e-17, -1e-18])
def test_growth_between_the_ends_is_refused(ctx, c):
    """p(1) = 0, but 30 s - 30 s^3 is 11.5 at s^2 = 1/3, and 45000 behind that."""
    from tenncor_amd import capi
    with pytest.raises(capi.TcgError, match="grow past"):
        run(ctx, gradient(8, 9), steps=4, coef=(30.0, -30.0, c))


@pytest.mark.parametrize("rows,cols", [(40, 56), (300, 200)])
@pytest.mark.parametrize("t", [np.float32, np.float64])
@pytest.mark.parametrize("steps,coef,top", [(2, (3.0, 2.0, 1.0), 8240), (1, (1.0, 0.0, 1e4), 10001), (2, (900.0, 0.0, 0.0), 810000)])
def test_values_below_a_million_after_the_last_step(ctx, rows, cols, t, steps, coef, top):
    """What another step would make of them does not matter."""
    from tenncor_amd import capi
    g = gradient(rows, cols, t, seed=22)
    close(run(ctx, g, steps=steps, coef=coef)[0], g[0], steps, coef)
    with pytest.raises(capi.TcgError, match="grow past"):
        run(ctx, g, steps=steps + 1, coef=coef)


# (rows, cols, batch): one workgroup, 64 x 64 tiles wide and tall, several matrices
@pytest.mark.parametrize("rows,cols,batch", [(1, 1, 1), (40, 56, 1), (300, 200, 1), (200, 310, 2), (5, 700, 3), (513, 777, 1)])
@pytest.mark.parametrize("steps,coef", [(1, (0.0, 1.0, 0.0)), (2, (0.0, 1.0, 0.0)), (3, (0.0, 1.0, 0.0)), (2, (0.0, 0.0, 1.0)),
                                        (3, (1e-7, 1.0, 0.5)), (2, (1e-6, -1.0, 2.0))])
def test_without_a_linear_term_worth_the_name(ctx, rows, cols, batch, steps, coef):
    """s -> s^3 three times is s^27: results far below the largest that any matrix could
    give.  Products in 64 bits, one rounding to float: 2^-24 of each element; in the norm
    2^-24 of the result's, and as much again for what the roundings in 64 bits come to
    (at most (8 + 777) sqrt(777) 2^-53 a step, taken up to 5 x 5 x 5 times by the steps:
    2^-31), and half of the smallest float an element."""
    g = gradient(rows, cols, batch=batch, seed=23)
    for pad, gap, shift, in_place in ((0, 0, 0, False), (3, 5, 1, True)):
        got = run(ctx, g, pad=pad, gap=gap, shift=shift, in_place=in_place, steps=steps, coef=coef)
        for z in range(batch):
            x = g[z].astype(np.float64)
            x = x / (np.linalg.norm(x) + 1e-7)
            for _ in range(steps):
                gram = x @ x.T
                x = coef[0] * x + (coef[1] * gram + coef[2] * (gram @ gram)) @ x
            off = np.linalg.norm(got[z].astype(np.float64) - x)
            assert off <= 1.01 * 2.0 ** -24 * np.linalg.norm(x) + 2.0 ** -150 * np.sqrt(rows * cols)
