"""Matrices side by side: column blocks of one wide matrix, as the gate matrices of a
recurrent cell lie in its fused weight."""
import numpy as np
import pytest

from test_gpu_orthogonalize import CODE, MARK, ctx, gradient, reference, run  # noqa: F401 (ctx is a fixture)

pytestmark = pytest.mark.gpu


def blocks(ctx, g, gap, pad, in_place, wide_in=True, wide_out=True):
    """g: [batch][rows][cols]; `gap` elements between blocks, `pad` behind the last."""
    t = g.dtype.type
    batch, rows, cols = g.shape
    stride = cols + gap
    ld = batch * stride - gap + pad

    def lay(v, wide):
        if not wide:
            return v.copy()
        host = np.full((rows, ld), MARK, t)
        for z in range(batch):
            host[:, z * stride:z * stride + cols] = v[z]
        return host

    src = ctx.upload(lay(g, wide_in))
    dst = src if in_place else ctx.upload(lay(np.zeros_like(g), wide_out))
    ctx.orthogonalize(CODE[t], rows, cols, batch, src.ptr, ld if wide_in else cols, stride if wide_in else rows * cols,
                      dst.ptr, ld if wide_out else cols, stride if wide_out else rows * cols)
    if not wide_out:
        return dst.get().reshape(g.shape)
    full = dst.get().reshape(rows, ld)
    out = np.stack([full[:, z * stride:z * stride + cols].copy() for z in range(batch)])
    for z in range(batch):
        full[:, z * stride:z * stride + cols] = MARK
    assert (full == MARK).all(), "wrote between the blocks"
    return out


@pytest.mark.parametrize("t", [np.float32, np.float64])
@pytest.mark.parametrize("batch,rows,cols", [(4, 64, 96), (3, 9, 5), (2, 200, 130), (2, 130, 203), (3, 1, 7), (2, 190, 2101)])
def test_column_blocks(ctx, batch, rows, cols, t):
    g = gradient(rows, cols, t, batch, seed=31)
    want = run(ctx, g)
    for gap, pad in ((0, 0), (3, 2)):
        np.testing.assert_array_equal(blocks(ctx, g, gap, pad, False), want)
        np.testing.assert_array_equal(blocks(ctx, g, gap, pad, True), want)
    np.testing.assert_array_equal(blocks(ctx, g, 1, 0, False, wide_in=False), want)
    np.testing.assert_array_equal(blocks(ctx, g, 1, 0, False, wide_out=False), want)


def test_matrices_that_do_overlap_are_refused(ctx):
    from tenncor_amd import capi
    a, b = ctx.upload(np.zeros(256, np.float32)), ctx.upload(np.zeros(256, np.float32))

    def call(ldi=12, stride_i=4, ldo=12, stride_o=4, rows=4, cols=4, batch=3):
        ctx.orthogonalize(2, rows, cols, batch, a.ptr, ldi, stride_i, b.ptr, ldo, stride_o)

    call()  # side by side: taken
    for args in ({"stride_i": 3}, {"stride_o": 3}, {"ldi": 11}, {"ldo": 11}, {"stride_i": 0}, {"ldi": 8, "stride_i": 12}):
        with pytest.raises(capi.TcgError, match="overlap"):
            call(**args)
    # distances whose sum wraps around, which would pass for small ones
    for args in ({"stride_i": 1 << 63}, {"stride_o": (1 << 64) - 4}, {"batch": 65535, "stride_o": (1 << 64) // 65534 + 1}):
        with pytest.raises(capi.TcgError, match="too far apart"):
            call(**args)
    ctx.sync()
    assert not a.get().any() and not b.get().any()


@pytest.mark.parametrize("tall", [False, True])
def test_offsets_past_32_bits(ctx, tall):
    """Two rows of 17 million: 2.2e9 halves of a padded X, 8.7e9 bytes.  Every sum of A runs over
    six additions in each of 2076 slabs (531250 shared by 256 workgroups): 0.25 sqrt(12456) =
    28 * 2^-24 in the mean, twice that is allowed; the other roundings, at most 12 * 2^-24 a step
    as derived in test_gpu_orthogonalize_kernels, count besides."""
    rng = np.random.default_rng(1)
    g = (rng.normal(0, 1, (2, 2)) @ rng.normal(0, 1, (2, 17_000_000))).astype(np.float32)
    want, size = reference(g, 2)
    got = run(ctx, (g.T.copy() if tall else g)[None], steps=2)[0]
    off = np.linalg.norm((got.T if tall else got) - want)
    assert off <= (56 + 12) * 2.0 ** -24 * size
