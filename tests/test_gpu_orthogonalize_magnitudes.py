"""tcg_orthogonalize at the ends of a type's range."""
import numpy as np
import pytest

from test_gpu_orthogonalize import close, ctx, gradient, run  # noqa: F401 (ctx is a fixture)

pytestmark = pytest.mark.gpu

SIZES = [(20, 30), (200, 150), (3, 5000)]


@pytest.mark.parametrize("rows,cols", SIZES)
def test_a_power_of_two_changes_nothing_in_double(ctx, rows, cols):
    """Squares beyond 2^1024 or below 2^-1074, and a norm beyond the largest double: without
    epsilon the same bits.  (Elements below 2^-100 would meet the others in another sum.)"""
    g = gradient(rows, cols, np.float64, seed=4, scale=1.0)
    g[abs(g) < 1e-6] = 0.0
    g /= 2.0 ** np.frexp(abs(g).max())[1]  # the largest element between 1/2 and 1
    want = run(ctx, g, eps=0.0)
    close(want[0], g[0], eps=0.0)
    for k in (-990, -900, -600, 600, 900, 1024):
        np.testing.assert_array_equal(run(ctx, np.ldexp(g, k), eps=0.0), want)


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("k", [-510, -505, -500, 498, 500, 505, 512])
def test_magnitudes_that_straddle_what_can_be_squared(ctx, rows, cols, k):
    """Some elements' squares are taken as they are and some scaled; the sums meet."""
    g = gradient(rows, cols, np.float64, seed=5, scale=1.0)
    close(run(ctx, np.ldexp(g, k), eps=0.0)[0], g[0], eps=0.0)


@pytest.mark.parametrize("rows,cols", SIZES)
def test_epsilon_beside_large_and_small_values(ctx, rows, cols):
    g = gradient(rows, cols, np.float64, seed=6, scale=1.0)
    for k, eps in ((600, 1e-7), (-600, np.ldexp(1.0, -599)), (700, np.ldexp(1.0, 702))):
        close(run(ctx, np.ldexp(g, k), eps=eps)[0], g[0], eps=np.ldexp(eps, -k))
    # next to an epsilon of usual size nothing is left of them
    assert abs(run(ctx, np.ldexp(g, -600), eps=1e-7)).max() < 1e-160


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("t", [np.float32, np.float64])
def test_a_matrix_of_zeros_stays_one_for_the_smallest_epsilon(ctx, rows, cols, t):
    for eps in (5e-324, 1e-310, 1e-300):
        assert not run(ctx, np.zeros((2, rows, cols), t), eps=eps).any()


@pytest.mark.parametrize("rows,cols", SIZES)
def test_values_that_are_none_among_large_ones(ctx, rows, cols):
    g = np.ldexp(gradient(rows, cols, np.float64, 3, seed=7, scale=1.0), 700)
    alone = run(ctx, g)
    for bad in (np.nan, np.inf, -np.inf):
        g[1, rows // 2, cols // 3] = bad
        got = run(ctx, g)
        assert np.isnan(got[1]).all()
        np.testing.assert_array_equal(got[[0, 2]], alone[[0, 2]])
