"""Every kernel that tcg_orthogonalize can choose, and a bound that the halves' smaller
terms matter to.

After five steps the tolerance of test_gpu_orthogonalize is 20 to 60 times what the
kernels are off by: it follows the worst case of every rounding through the largest
slopes.  Here two steps are taken of matrices with six strong directions, and the
roundings are counted as what they are, independent of each other, with their mean
square: relative to what it rounds, the second half leaves 2^-24.4 (the first one's
rest is even over half a step of its own, the second one's step follows that rest),
six operands a step; the sums of A, the longest, run over 3 n / 16 additions, whose
errors of at most 2^-24 of a partial sum, 0.29 * 1.5 of that in the mean, come to
sqrt(n / 16) 0.44 2^-24 <= 7 * 2^-24 at 4200 columns; a, b and c weigh them by at most
one where all six directions are of size 0.4.  Together below 2.5 * 2^-22 of the
iterate a step, and 3 * 2^-22 is allowed, times the slopes as there.  The last test
here plants the loss of one of the smaller terms of a product into a computation on
the CPU and finds it outside.
"""
import numpy as np
import pytest

from test_gpu_orthogonalize import COEF, close, ctx, gradient, reference, run  # noqa: F401 (ctx is a fixture)

ETA = 3 * 2.0 ** -22


def strong(rows, cols, seed=0):
    rng = np.random.default_rng(seed)
    rank = min(6, rows, cols)
    g = rng.normal(0, 1, (rows, rank)) @ rng.normal(0, 1, (rank, cols)) + 1e-3 * rng.normal(0, 1, (rows, cols))
    return (1e-3 * g).astype(np.float32)


def share(got, g, steps=2):
    """The distance from the iteration in 64 bits, as a share of what is allowed."""
    want, size = reference(g, steps)
    return np.linalg.norm(got.astype(np.float64) - want) / (ETA * size)


# in one workgroup with one and with two tiles a wave, for every number of tiles along the short side;
# tiles of 64 with and without others to share A with; A in 128 and the rest in 192; all in 128; all in 192
TWO_STEPS = [(20, 300), (20, 1000), (1000, 31), (64, 96), (60, 500), (90, 120), (90, 310), (310, 95), (128, 130), (125, 160),
             (513, 777), (640, 384), (260, 3100), (3100, 250), (1500, 1600), (1600, 1500), (2000, 2050), (2050, 2000), (2100, 2200), (2200, 2100)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", TWO_STEPS)
def test_two_steps(ctx, rows, cols):
    g = strong(rows, cols, rows)
    got = share(run(ctx, g[None], pad=1, steps=2)[0], g)
    assert got <= 1, got


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(4100, 4150), (4200, 4100)])
def test_tiles_of_192_for_every_product(ctx, rows, cols):
    """4160 padded rows are 21 tiles and two thirds of one; wide and tall."""
    g = strong(rows, cols, 7)
    got = share(run(ctx, g[None], steps=2)[0], g)
    assert got <= 1, got


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(530, 4000), (4000, 530), (2000, 2050)])
def test_double_in_tiles_of_64(ctx, rows, cols):
    """512 tiles of 64 x 64 and more: in the product with the iterate, and (2000 rows) in A and B."""
    g = gradient(rows, cols, np.float64, seed=8)
    close(run(ctx, g, pad=1)[0], g[0])


@pytest.mark.gpu
@pytest.mark.parametrize("batch,rows,cols", [(9, 400, 520), (9, 520, 400)])
def test_several_in_double_in_tiles_of_64(ctx, batch, rows, cols):
    g = gradient(rows, cols, np.float64, batch, seed=9)
    got = run(ctx, g, gap=7)
    for z in (0, 4, 8):
        close(got[z], g[z])
        np.testing.assert_array_equal(run(ctx, g, gap=7)[z], got[z])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,cut", [(770, 800, 4), (2000, 2050, 6), (4096, 4096, 9)])
def test_the_sums_of_the_last_product_are_cut(ctx, rows, cols, cut):
    """Rows that are all the same: the addends of an element of B X are too, and the roundings
    of a long sum fall to one side as long as it does not double.  Sums of `cut` slabs of six
    additions and their sum in turn are off by at most (3 cut + slabs / cut / 2) 2^-24 (an
    addition by 2^-24 of the sum so far, half of the last one on the way); the halves of B
    and X leave 2^-24.4 each in the mean, the sum with a X, its product with the scale and
    the rounding of X at most 2^-24 each: 5 together.  (One sum over all slabs comes to 10, 27 and 55 * 2^-24 here, in
    an emulation of its additions, beside 2 to 4.5 of sums that are cut: a third of the first
    bound is asked for, which is the mean of errors that are even between it and zero.)
    Errors of A are the same for all elements, as A has one value, and fall to the factor
    between the result and the matrix, which is taken out."""
    rng = np.random.default_rng(3)
    v = rng.uniform(0.5, 1, cols).astype(np.float32)
    got = run(ctx, np.repeat(v[None] * np.float32(1e-3), rows, 0)[None], steps=1, coef=(0.01, 1.0, 0.0), eps=0.0)[0].astype(np.float64)
    v = (v * np.float32(1e-3)).astype(np.float64)
    slabs = -(-(-(-rows // 64) * 64) // 32)
    factor = (got @ v).mean() / (v @ v)
    off = np.linalg.norm(got - factor * v) / (factor * np.sqrt(rows) * np.linalg.norm(v))
    assert off <= ((3 * cut + slabs / cut / 2) / 3 + 5) * 2.0 ** -24, off * 2.0 ** 24


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(530, 4000), (4000, 530)])
def test_floats_in_double_in_tiles_of_64(ctx, rows, cols):
    """s -> s^9, whose products are in double: one rounding to float, 2^-24 of the result, and a
    hundredth of it for what those in double come to (9 (8 + 4000) sqrt(530) 2^-53 = 2^-33)."""
    g = gradient(rows, cols, seed=10)
    got = run(ctx, g, pad=1, steps=2, coef=(0.0, 1.0, 0.0))[0].astype(np.float64)
    x = g[0].astype(np.float64).T if rows > cols else g[0].astype(np.float64)
    x = x / (np.linalg.norm(x) + 1e-7)
    for _ in range(2):
        x = (x @ x.T) @ x
    x = x.T if rows > cols else x
    assert np.linalg.norm(got - x) <= 1.01 * 2.0 ** -24 * np.linalg.norm(x)


# ---- the bound itself ---------------------------------------------------------------

def halves(x, top):
    scale = 2.0 ** (15 - np.frexp(top)[1])
    v = (x * scale).astype(np.float32)
    hi = v.astype(np.float16).astype(np.float32)
    return hi.astype(np.float64) / scale, (v - hi).astype(np.float16).astype(np.float64) / scale


def product(p, q, lost):
    """p q^T of two split matrices"""
    out = p[0] @ q[0].T
    for name, part in (("hi lo", (p[0], q[1])), ("lo hi", (p[1], q[0]))):
        if name != lost:
            out = out + part[0] @ part[1].T
    return out


def emulated(g, steps, lost=(None, None, None)):
    """The iteration over split operands with exact sums, without the products `lost` of A, A A and B X."""
    a, b, c = COEF
    x = g.astype(np.float64)
    x = x / (np.linalg.norm(x) + 1e-7)
    tall = x.shape[0] > x.shape[1]
    x = (x.T if tall else x).astype(np.float32).astype(np.float64)
    top = 1.0001
    for _ in range(steps):
        xs = halves(x, top)
        gram = product(xs, xs, lost[0]).astype(np.float32)
        grams = halves(gram, top * top)
        factor = (b * gram + c * product(grams, grams, lost[1])).astype(np.float32)
        s = np.linspace(0, top, 4001)
        factors = halves(factor, abs(b * s ** 2 + c * s ** 4).max() * 1.0001)
        x = (a * x + product(factors, halves(x.T, top), lost[2])).astype(np.float32).astype(np.float64)
        top = abs(s * (a + b * s ** 2 + c * s ** 4)).max() * 1.0001
    return x.T if tall else x


@pytest.mark.parametrize("rows,cols", [(20, 300), (64, 96), (310, 95), (513, 777), (640, 384), (260, 3100)])
def test_the_bound_notices_a_lost_product(rows, cols):
    g = strong(rows, cols, rows)
    assert share(emulated(g, 2), g) <= 0.5
    for lost in (("hi lo", None, None), (None, "lo hi", None), (None, None, "hi lo"), (None, None, "lo hi")):
        assert share(emulated(g, 2, lost), g) > 1.5, lost
