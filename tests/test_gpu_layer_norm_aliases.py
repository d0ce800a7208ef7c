"""tcg_layer_norm_grad with dweight or dbias in the place of the weight: the weight is
read before they are written, on every route."""
import numpy as np
import pytest

from test_gpu_layer_norm import CODE, ctx, data, reference  # noqa: F401 (ctx is a fixture)

pytestmark = pytest.mark.gpu


# one launch for all gradients, two launches, rows beyond registers
@pytest.mark.parametrize("rows,cols", [(300, 64), (256, 512), (700, 1500), (2000, 300), (20, 9000), (40, 40000)])
@pytest.mark.parametrize("t", [np.float32, np.float64])
@pytest.mark.parametrize("given", [False, True])
def test_gradients_in_the_place_of_the_weight(ctx, rows, cols, t, given):
    x, w, b, g = data(rows, cols, t, rows)
    full = reference(x, w, b, 1e-5)
    bx, bg = ctx.upload(x), ctx.upload(g)
    mean, rstd = (ctx.upload(full[k].astype(t)) if given else None for k in ("mean", "rstd"))

    def grads(where):
        weight = ctx.upload(w)
        out = {k: ctx.upload(np.zeros(n, t)) for k, n in (("dx", rows * cols), ("dw", cols), ("db", cols))}
        if where:
            out[where] = weight
        ctx.layer_norm_grad(CODE[t], rows, cols, bg.ptr, cols, bx.ptr, cols, weight.ptr, 1e-5, dx=out["dx"].ptr, lddx=cols,
                            dweight=out["dw"].ptr, dbias=out["db"].ptr, mean=mean and mean.ptr, rstd=rstd and rstd.ptr)
        return {k: v.get() for k, v in out.items()}

    want = reference(x, w, b, 1e-5, g, full["mean"].astype(t), full["rstd"].astype(t)) if given else reference(x, w, b, 1e-5, g)
    apart = grads(None)
    for where in ("dw", "db"):
        got = grads(where)
        for k in got:
            # another route may add up in another order, within the operator's tolerance
            off = abs(got[k].astype(np.longdouble).reshape(want[k].shape) - want[k])
            u = 2.0 ** -24 if t == np.float32 else 2.0 ** -53
            assert (off <= 300 * u * want[k + "_size"]).all(), (where, k)
        np.testing.assert_array_equal(got["dx"], apart["dx"])
