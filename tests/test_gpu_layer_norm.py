"""tcg_layer_norm and tcg_layer_norm_grad against the formulas in 64 bits, and
LAYER_NORM nodes in graphs.

Tolerances.  u = eps / 2 of the type is the largest relative error of one
rounding.  A row's sums run over at most 64 elements a lane (chunks of long rows
are joined in double), six halvings of a wave and 16 waves: a sum of
non-negative terms is off by at most 90 u of itself, any sum by at most 90 u of
the sum of the terms' magnitudes.

  r: half of 90 u and a division and a root -> 50 u
  h = ((x - m) - c) r: the two differences 2 u of |x - m|; c's own error 90 u of
     mean|d| <= 1 / r, so 90 u of h's unit; r 50 u -> 150 u (|h| + 1)
  y = h w + b: 150 u (|h| + 1) |w| and two more roundings -> 160 u ((|h| + 1) |w| + |b|)
  dx = r (g w - mean(g w) - h mean(g w h)): every factor above at most once:
     300 u r (|g w| + mean|g w| + (|h| + 1) mean|g w| + (|h| + 1) mean(|g w| (|h| + 1)))
  dw: h's error and the order of the sum over rows (at most 128 partial sums on
     the way of a term, see the launches): 300 u sum |g| (|h| + 1); db: 150 u sum |g|
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}
CODE = {np.float32: 2, np.float64: 1}


@pytest.fixture(scope="module")
def ctx():
    from tenncor_amd import capi
    c = capi.Context(0)
    yield c
    c.close()


def wide(t):
    """The formulas' type: 64 bits, or more where the operands have 64."""
    return np.float64 if t == np.float32 else np.longdouble


def reference(x, w, b, eps, g=None, mean=None, rstd=None):
    """y, mean, rstd and, for the gradient g, dx, dw, db with the tolerances' magnitudes."""
    f = wide(x.dtype.type)
    x, w, b = x.astype(f), w.astype(f), b.astype(f)
    m = x.mean(1, keepdims=True) if mean is None else mean.astype(f)[:, None]
    r = 1 / np.sqrt(((x - m) ** 2).mean(1, keepdims=True) + f(eps)) if rstd is None else rstd.astype(f)[:, None]
    h = (x - m) * r
    out = {"y": h * w + b, "mean": m[:, 0], "rstd": r[:, 0], "y_size": (abs(h) + 1) * abs(w) + abs(b)}
    if g is not None:
        g = g.astype(f)
        gw, big = g * w, abs(h) + 1
        av = lambda v: v.mean(1, keepdims=True)  # noqa: E731
        out["dx"] = r * (gw - av(gw) - h * av(gw * h))
        out["dx_size"] = r * (abs(gw) + av(abs(gw)) + big * av(abs(gw)) + big * av(abs(gw) * big))
        out["dw"], out["dw_size"] = (g * h).sum(0), (abs(g) * big).sum(0)
        out["db"], out["db_size"] = g.sum(0), abs(g).sum(0)
    return out


def close(got, want, size, steps, t):
    off = abs(got.astype(np.longdouble) - want)
    assert got.shape == want.shape and not np.isnan(got).any()
    assert (off <= steps * U[t] * size).all(), "off by %g of the tolerance" % float((off / (steps * U[t] * size)).max())


class Rows:
    """A matrix on the device with `pad` elements of a known value between its rows."""

    MARK = -77.0

    def __init__(self, ctx, data, pad, shift=0):
        self.ctx, self.pad, self.shift = ctx, pad, shift
        self.rows, self.cols = data.shape
        self.ld = self.cols + pad
        full = np.full((self.rows, self.ld), self.MARK, data.dtype)
        full[:, :self.cols] = data
        self.host = np.concatenate([np.full(shift, self.MARK, data.dtype), full.reshape(-1)])
        self.buf = ctx.upload(self.host)
        self.ptr = self.buf.ptr + shift * data.dtype.itemsize

    def get(self):
        """The rows; whatever lies between them has stayed as it was."""
        flat = self.buf.get()
        assert (flat[:self.shift] == self.MARK).all()
        full = flat[self.shift:].reshape(self.rows, self.ld)
        assert (full[:, self.cols:] == self.MARK).all()
        return full[:, :self.cols]


def data(rows, cols, t, seed, offset=0.0):
    rng = np.random.default_rng(seed)
    x = (rng.normal(0, 1, (rows, cols)) * rng.uniform(0.1, 3, (rows, 1)) + rng.normal(0, 1, (rows, 1)) + offset).astype(t)
    return x, rng.normal(1, 0.2, cols).astype(t), rng.normal(0, 1, cols).astype(t), rng.normal(0, 1, (rows, cols)).astype(t)


def run_forward(ctx, x, w, b, eps, pad=0, shift=0, stats=True):
    t = x.dtype.type
    dx = Rows(ctx, x, pad, shift)
    dy = Rows(ctx, np.zeros_like(x), pad, shift)
    dw, db = (None if v is None else Rows(ctx, v[None], 0, shift) for v in (w, b))
    mean, rstd = (ctx.empty(len(x), t) if stats else None for _ in range(2))
    ctx.layer_norm(CODE[t], len(x), x.shape[1], dx.ptr, dx.ld, dw and dw.ptr, db and db.ptr, eps, dy.ptr, dy.ld,
                   mean and mean.ptr, rstd and rstd.ptr)
    return dy.get(), mean and mean.get(), rstd and rstd.get()


def run_backward(ctx, g, x, w, eps, stats=None, pad=0, shift=0, want=("dx", "dw", "db")):
    t = x.dtype.type
    rows, cols = x.shape
    dg, dxin = Rows(ctx, g, pad, shift), Rows(ctx, x, 2 * pad, shift)
    dw = None if w is None else Rows(ctx, w[None], 0, shift)
    kept = [ctx.upload(s) for s in stats] if stats is not None else [None, None]
    outs = {"dx": Rows(ctx, np.zeros_like(x), pad, shift), "dw": Rows(ctx, np.zeros((1, cols), t), 0, shift),
            "db": Rows(ctx, np.zeros((1, cols), t), 0, shift)}
    ptr = {k: outs[k].ptr if k in want else None for k in outs}
    ctx.layer_norm_grad(CODE[t], rows, cols, dg.ptr, dg.ld, dxin.ptr, dxin.ld, dw and dw.ptr, eps, dx=ptr["dx"],
                        lddx=outs["dx"].ld, dweight=ptr["dw"], dbias=ptr["db"], mean=kept[0] and kept[0].ptr, rstd=kept[1] and kept[1].ptr)
    return {k: v.get() if k == "dx" else v.get()[0] for k, v in outs.items()}


# one to many lanes, waves and registers a row; odd lengths; rows that leave the last workgroup half empty;
# the last lengths that fit registers and the first that do not
SIZES = [(1, 1), (3, 1), (1, 7), (5, 2), (7, 63), (9, 64), (4, 255), (33, 256), (6, 257), (5, 512), (3, 1000), (130, 1023),
         (5, 1025), (3, 2047), (4, 2048), (2, 2049), (3, 4096), (2, 4099), (2, 8191), (2, 8193), (2, 16384), (3, 16385), (1, 20001),
         (2, 32768), (2, 32769), (3, 100003)]


@pytest.mark.parametrize("t", [np.float32, np.float64])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_forward(ctx, rows, cols, t):
    x, w, b, _ = data(rows, cols, t, rows * 100003 + cols)
    for pad, shift in ((0, 0), (3, 1)):
        y, mean, rstd = run_forward(ctx, x, w, b, 1e-5, pad, shift)
        want = reference(x, w, b, 1e-5)
        close(y, want["y"], want["y_size"], 160, t)
        close(mean, want["mean"], abs(want["mean"]) + 90 / want["rstd"], 2, t)
        close(rstd, want["rstd"], want["rstd"], 50, t)
        bare, _, _ = run_forward(ctx, x, None, None, 1e-5, pad, shift, stats=False)
        plain = reference(x, np.ones_like(w), np.zeros_like(b), 1e-5)
        close(bare, plain["y"], plain["y_size"], 160, t)


@pytest.mark.parametrize("t", [np.float32, np.float64])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_gradients(ctx, rows, cols, t):
    x, w, b, g = data(rows, cols, t, rows * 7 + cols)
    for pad, shift, given in ((0, 0, False), (3, 1, True)):
        stats = None
        if given:
            full = reference(x, w, b, 1e-5)
            stats = [full["mean"].astype(t), full["rstd"].astype(t)]
        want = reference(x, w, b, 1e-5, g, *(stats or [None, None]))
        got = run_backward(ctx, g, x, w, 1e-5, stats, pad, shift)
        close(got["dx"], want["dx"], want["dx_size"], 300, t)
        close(got["dw"], want["dw"], want["dw_size"], 300, t)
        close(got["db"], want["db"], want["db_size"], 150, t)


@pytest.mark.parametrize("rows,cols", [(1200, 96), (5003, 130), (20000, 40), (3000, 1100), (2500, 4100), (40, 40000)])
def test_sums_over_many_rows(ctx, rows, cols):
    """More rows than one sweep of the grid, all three gradients and each alone, the same bits twice."""
    t = np.float32
    x, w, b, g = data(rows, cols, t, 5)
    want = reference(x, w, b, 1e-5, g)
    got = run_backward(ctx, g, x, w, 1e-5)
    close(got["dx"], want["dx"], want["dx_size"], 300, t)
    close(got["dw"], want["dw"], want["dw_size"], 300, t)
    close(got["db"], want["db"], want["db_size"], 150, t)
    again = run_backward(ctx, g, x, w, 1e-5)
    for k in got:
        np.testing.assert_array_equal(got[k], again[k])
    for k in got:
        alone = run_backward(ctx, g, x, w, 1e-5, want=(k,))
        close(alone[k], want[k], want[k + "_size"], 300, t)
        for other in got:
            assert other == k or not alone[other].any(), "wrote a gradient that was not wanted"


@pytest.mark.parametrize("t", [np.float32, np.float64])
@pytest.mark.parametrize("rows", [1, 63, 64, 65, 129, 700, 768, 769, 1500])
@pytest.mark.parametrize("cols", [1, 3, 4, 30, 64, 130, 515, 1100, 4096, 4100])
def test_all_gradients_with_known_statistics(ctx, rows, cols, t):
    """Few rows take one launch for all gradients, more rows two; the same bits at every call."""
    x, w, b, g = data(rows, cols, t, rows + cols)
    full = reference(x, w, b, 1e-5)
    stats = [full["mean"].astype(t), full["rstd"].astype(t)]
    want = reference(x, w, b, 1e-5, g, *stats)
    for names in (("dx", "dw", "db"), ("dx", "dw"), ("dx", "db")):
        got = run_backward(ctx, g, x, w, 1e-5, stats, pad=1, shift=1, want=names)
        for k, ops in (("dx", 300), ("dw", 300), ("db", 150)):
            if k in names:
                close(got[k], want[k], want[k + "_size"], ops, t)
            else:
                assert not got[k].any(), "wrote a gradient that was not wanted"
        again = run_backward(ctx, g, x, w, 1e-5, stats, pad=1, shift=1, want=names)
        for k in got:
            np.testing.assert_array_equal(got[k], again[k])


@pytest.mark.parametrize("rows,cols,t", [(400000, 60, np.float32), (70000, 331, np.float32), (6000, 4099, np.float32), (9000, 1300, np.float64)])
def test_more_than_the_caches_hold(ctx, rows, cols, t):
    """Rows of every shape of the kernels, with 280 MB of x, g and dx.  The longest chain of a sum over rows: 49."""
    x, w, b, g = data(rows, cols, t, 6)
    want = reference(x, w, b, 1e-5, g)
    got = run_backward(ctx, g, x, w, 1e-5, pad=1)
    close(got["dx"], want["dx"], want["dx_size"], 300, t)
    close(got["dw"], want["dw"], want["dw_size"], 300, t)
    close(got["db"], want["db"], want["db_size"], 150, t)


@pytest.mark.parametrize("t", [np.float32, np.float64])
@pytest.mark.parametrize("cols", [5, 300, 5000, 40000])
def test_rows_far_from_zero(ctx, cols, t):
    """The mean's own rounding is taken out: an offset of 4096 deviations costs nothing but
    the input's own bits."""
    x, w, b, g = data(6, cols, t, 3)
    x = (x.astype(np.float64) * 0.25 + 4096).astype(t)
    want = reference(x, w, b, 1e-5, g)
    y, _, _ = run_forward(ctx, x, w, b, 1e-5)
    close(y, want["y"], want["y_size"], 160, t)
    got = run_backward(ctx, g, x, w, 1e-5)
    close(got["dx"], want["dx"], want["dx_size"], 300, t)
    close(got["dw"], want["dw"], want["dw_size"], 300, t)


@pytest.mark.parametrize("cols", [1, 6, 300, 2500, 17000, 40000])
def test_rows_without_spread_and_values_that_are_none(ctx, cols):
    t = np.float32
    x, w, b, g = data(5, cols, t, 9)
    x[1] = 2.5                 # equal elements: the bias, whatever epsilon above zero
    x[2, cols // 2] = np.nan   # stays in its row
    x[3, cols - 1] = np.inf
    y, mean, rstd = run_forward(ctx, x, w, b, 1e-5)
    np.testing.assert_array_equal(y[1], b)
    assert np.isnan(y[2]).all() and np.isnan(y[3]).all()
    assert mean[3] == np.inf and np.isnan(mean[2]) and mean[1] == 2.5
    sound = [0, 4]
    want = reference(x[sound], w, b, 1e-5, g[sound])
    close(y[sound], want["y"], want["y_size"], 160, t)
    got = run_backward(ctx, g, x, w, 1e-5)
    close(got["dx"][sound], want["dx"], want["dx_size"], 300, t)
    assert np.isnan(got["dx"][2]).all() and np.isnan(got["dx"][3]).all()
    assert np.isnan(got["dw"]).all()
    close(got["db"], g.astype(np.float64).sum(0), abs(g.astype(np.float64)).sum(0), 150, t)
    # epsilon zero: 0 / 0 in the row of equal elements, nothing elsewhere
    y0, _, _ = run_forward(ctx, x, w, b, 0.0)
    assert np.isnan(y0[1]).all() and (cols == 1 or not np.isnan(y0[sound]).any())


@pytest.mark.parametrize("rows,cols", [(300, 64), (20, 1500), (9, 9000), (3, 40000)])
def test_in_place(ctx, rows, cols):
    t = np.float32
    x, w, b, g = data(rows, cols, t, 13)
    want, _, _ = run_forward(ctx, x, w, b, 1e-5)
    dx, dw, db = ctx.upload(x), ctx.upload(w), ctx.upload(b)
    ctx.layer_norm(CODE[t], rows, cols, dx.ptr, cols, dw.ptr, db.ptr, 1e-5, dx.ptr, cols)
    np.testing.assert_array_equal(dx.get().reshape(rows, cols), want)
    grads = run_backward(ctx, g, x, w, 1e-5)
    for where in ("dy", "x"):
        bx, bg, ow, ob = ctx.upload(x), ctx.upload(g), ctx.empty(cols, t), ctx.empty(cols, t)
        out = bg if where == "dy" else bx
        ctx.layer_norm_grad(CODE[t], rows, cols, bg.ptr, cols, bx.ptr, cols, dw.ptr, 1e-5, dx=out.ptr, lddx=cols,
                            dweight=ow.ptr, dbias=ob.ptr)
        np.testing.assert_array_equal(out.get().reshape(rows, cols), grads["dx"])
        np.testing.assert_array_equal(ow.get(), grads["dw"])
        np.testing.assert_array_equal(ob.get(), grads["db"])


@pytest.mark.parametrize("rows,cols", [(300, 64), (20, 1500)])
def test_in_place_with_known_statistics(ctx, rows, cols):
    """dx over dy or x: the sums over rows have read both before."""
    t = np.float32
    x, w, b, g = data(rows, cols, t, 14)
    full = reference(x, w, b, 1e-5)
    stats = [full["mean"].astype(t), full["rstd"].astype(t)]
    want = reference(x, w, b, 1e-5, g, *stats)
    for where in ("dy", "x"):
        bx, bg, bw, bm, br, ow, ob = (ctx.upload(v) for v in (x, g, w, *stats, w, w))
        out = bg if where == "dy" else bx
        ctx.layer_norm_grad(CODE[t], rows, cols, bg.ptr, cols, bx.ptr, cols, bw.ptr, 1e-5, dx=out.ptr, lddx=cols,
                            dweight=ow.ptr, dbias=ob.ptr, mean=bm.ptr, rstd=br.ptr)
        close(out.get().reshape(rows, cols), want["dx"], want["dx_size"], 300, t)
        close(ow.get(), want["dw"], want["dw_size"], 300, t)
        close(ob.get(), want["db"], want["db_size"], 150, t)


def test_no_rows(ctx):
    one = ctx.upload(np.ones(8, np.float32))
    ctx.layer_norm(2, 0, 8, None, 8, one.ptr, one.ptr, 1e-5, None, 8)
    dw, db = ctx.upload(np.ones(8, np.float32)), ctx.upload(np.ones(8, np.float32))
    ctx.layer_norm_grad(2, 0, 8, None, 8, None, 8, one.ptr, 1e-5, dweight=dw.ptr, dbias=db.ptr)
    assert not dw.get().any() and not db.get().any()


def test_refusals(ctx):
    from tenncor_amd import capi
    a, b = ctx.upload(np.zeros(64, np.float32)), ctx.upload(np.zeros(64, np.float32))

    def forward(dtype=2, rows=4, cols=8, x=a.ptr, ldx=8, eps=1e-5, y=b.ptr, ldy=8, mean=None, rstd=None):
        ctx.layer_norm(dtype, rows, cols, x, ldx, None, None, eps, y, ldy, mean, rstd)

    def backward(dtype=2, rows=4, cols=8, dy=a.ptr, lddy=8, x=b.ptr, ldx=8, eps=1e-5, dx=None, lddx=8, dweight=a.ptr, mean=None):
        ctx.layer_norm_grad(dtype, rows, cols, dy, lddy, x, ldx, None, eps, dx=dx, lddx=lddx, dweight=dweight, mean=mean)

    for call, args, match in [
            (forward, {"dtype": 3}, "neither float nor double"), (forward, {"cols": 0}, "no elements"),
            (forward, {"ldx": 7}, "leading dims"), (forward, {"ldy": 7}, "leading dims"), (forward, {"eps": -1.0}, "eps"),
            (forward, {"eps": float("nan")}, "eps"), (forward, {"x": None}, "NULL"), (forward, {"y": None}, "NULL"),
            (forward, {"mean": a.ptr}, "together"), (forward, {"rstd": a.ptr}, "together"),
            (forward, {"y": a.ptr, "ldy": 9}, "in place"), (forward, {"rows": 1 << 62}, "too many"),
            (backward, {"dtype": 10}, "neither float nor double"), (backward, {"cols": 0}, "no elements"),
            (backward, {"lddy": 7}, "leading dims"), (backward, {"ldx": 7}, "leading dims"),
            (backward, {"dx": a.ptr, "lddx": 7}, "leading dims"), (backward, {"eps": -1.0}, "eps"),
            (backward, {"mean": a.ptr}, "together"), (backward, {"dweight": None}, "no gradient"), (backward, {"x": None}, "NULL"),
            (backward, {"dx": a.ptr, "lddx": 9}, "in place"), (backward, {"rows": 1 << 62}, "too many")]:
        with pytest.raises(capi.TcgError, match=match):
            call(**args)
    ctx.sync()
    assert not a.get().any() and not b.get().any()


def test_recorded_and_replayed(ctx):
    """Two recordings whose temporaries are their own, replayed in turn between eager calls."""
    t = np.float32
    cases = []
    for rows, cols in ((70, 200), (3, 40000)):
        x, w, b, g = data(rows, cols, t, cols)
        bufs = [ctx.upload(v) for v in (x, w, b, g)]
        outs = [ctx.empty(n, t) for n in (rows * cols, rows * cols, cols, cols)]

        def calls(bufs=bufs, outs=outs, rows=rows, cols=cols):
            bx, bw, bb, bg = (v.ptr for v in bufs)
            ctx.layer_norm(2, rows, cols, bx, cols, bw, bb, 1e-5, outs[0].ptr, cols)
            ctx.layer_norm_grad(2, rows, cols, bg, cols, bx, cols, bw, 1e-5, dx=outs[1].ptr, lddx=cols, dweight=outs[2].ptr, dbias=outs[3].ptr)

        calls()
        want = [o.get() for o in outs]
        ctx.capture_begin()
        calls()
        cases.append((ctx.capture_end(), bufs, outs, want, calls, (rows, cols)))
    for turn in range(3):
        for graph, bufs, outs, want, calls, (rows, cols) in cases:
            ctx.ew_unary("NEG", 2, rows * cols, bufs[0].ptr, bufs[0].ptr)
            calls()  # eager, on the negated rows
            ctx.sync()
            ctx.ew_unary("NEG", 2, rows * cols, bufs[0].ptr, bufs[0].ptr)
            for o in outs:
                ctx.fill_zero(o.ptr, o.nbytes)
        for graph, *_ in cases:
            ctx.graph_launch(graph)
        for graph, bufs, outs, want, calls, _ in cases:
            for o, v in zip(outs, want):
                np.testing.assert_array_equal(o.get(), v)
    for graph, *_ in cases:
        ctx.graph_destroy(graph)


def test_in_a_batch_and_beside_a_fork(ctx):
    """Inside tcg_batch_begin the steps held back go out first; on the forked stream the
    temporaries are kept until the join."""
    t = np.float32
    rows, cols = 40, 96
    x, w, b, g = data(rows, cols, t, 2)
    want, _, _ = run_forward(ctx, -x, w, b, 1e-5)
    bx, bw, bb, bg, neg, y = (ctx.upload(v) for v in (x, w, b, g, np.zeros_like(x), np.zeros_like(x)))
    ctx.batch_begin()
    ctx.ew_unary("NEG", 2, rows * cols, bx.ptr, neg.ptr)
    ctx.layer_norm(2, rows, cols, neg.ptr, cols, bw.ptr, bb.ptr, 1e-5, y.ptr, cols)
    ctx.batch_end()
    np.testing.assert_array_equal(y.get().reshape(rows, cols), want)
    grads = run_backward(ctx, g, x, w, 1e-5)
    outs = [ctx.upload(np.zeros(n, t)) for n in (rows * cols, cols, cols)]
    side = [ctx.upload(np.zeros(n, t)) for n in (rows * cols, cols, cols)]
    ctx.fork()
    ctx.layer_norm_grad(2, rows, cols, bg.ptr, cols, bx.ptr, cols, bw.ptr, 1e-5, dx=side[0].ptr, lddx=cols, dweight=side[1].ptr, dbias=side[2].ptr)
    ctx.fork_end()
    ctx.layer_norm_grad(2, rows, cols, bg.ptr, cols, bx.ptr, cols, bw.ptr, 1e-5, dx=outs[0].ptr, lddx=cols, dweight=outs[1].ptr, dbias=outs[2].ptr)
    ctx.join()
    for o, s, k in zip(outs, side, ("dx", "dw", "db")):
        np.testing.assert_array_equal(o.get(), grads[k].reshape(-1))
        np.testing.assert_array_equal(s.get(), grads[k].reshape(-1))


def test_a_recording_as_one_kernel_declines(ctx):
    from tenncor_amd import capi
    a = ctx.upload(np.zeros(64, np.float32))
    ctx.capture_begin(small=True)
    with pytest.raises(capi.TcgError) as err:
        ctx.layer_norm(2, 4, 16, a.ptr, 16, None, None, 1e-5, a.ptr, 16)
    assert err.value.status == 3
    ctx.capture_abort()


def test_an_offset_past_32_bits(ctx):
    """Rows far apart: element offsets beyond 2^32 (the last row starts 4.3e9 elements in)."""
    t = np.float32
    rows, cols = 3, 40
    ld = (1 << 31) + 8
    x, w, b, g = data(rows, cols, t, 1)
    base = ctx.alloc(4 * (2 * ld + cols))
    try:
        for i in range(rows):
            ctx.h2d(base + 4 * i * ld, x[i])
        y = ctx.empty(rows * cols, t)
        ctx.layer_norm(2, rows, cols, base, ld, None, None, 1e-5, y.ptr, cols)
        np.testing.assert_array_equal(y.get().reshape(rows, cols), run_forward(ctx, x, None, None, 1e-5)[0])
        bg, dw = ctx.upload(g), ctx.empty(cols, t)
        ctx.layer_norm_grad(2, rows, cols, bg.ptr, cols, base, ld, None, 1e-5, dx=y.ptr, lddx=cols, dweight=dw.ptr)
        want = run_backward(ctx, g, x, None, 1e-5)
        np.testing.assert_array_equal(y.get().reshape(rows, cols), want["dx"])
        np.testing.assert_array_equal(dw.get(), want["dw"])
    finally:
        ctx.free(base, 4 * (2 * ld + cols))


def test_ops(ctx):
    from tenncor_amd import ops
    t = np.float32
    x, w, b, g = data(6, 35, t, 4)
    tx, tw, tb, tg = ops.from_host(ctx, x, [5, 7, 3, 2]), ops.from_host(ctx, w, [5, 7]), ops.from_host(ctx, b, [5, 7]), ops.from_host(ctx, g, [5, 7, 3, 2])
    y, mean, rstd = ops.layer_norm(tx, tw, tb, ndims=2, stats=True)
    assert mean.shape == [1, 1, 3, 2, 1, 1, 1, 1]
    want = reference(x, w, b, 1e-5, g)
    close(y.get().reshape(6, 35), want["y"], want["y_size"], 160, t)
    dx, dw, db = ops.layer_norm_grad(tg, tx, tw, ndims=2)
    close(dx.get().reshape(6, 35), want["dx"], want["dx_size"], 300, t)
    close(dw.get(), want["dw"], want["dw_size"], 300, t)
    kept = reference(x, w, b, 1e-5, g, mean.get(), rstd.get())
    dx, dw, db = ops.layer_norm_grad(tg, tx, tw, ndims=2, mean=mean, rstd=rstd)
    close(dx.get().reshape(6, 35), kept["dx"], kept["dx_size"], 300, t)
    close(db.get(), want["db"], want["db_size"], 150, t)


# ---- in graphs ------------------------------------------------------------------

def layer_graph(g, api, t, seed=0, shape=(12, 5, 3), ndims=1):
    rng = np.random.default_rng(seed)
    head = list(shape[:ndims])
    x = g.variable(rng.normal(0.5, 1, int(np.prod(shape))).astype(t), list(shape), "x")
    w = g.variable(rng.normal(1, 0.2, int(np.prod(head))).astype(t), head, "w")
    b = g.variable(rng.normal(0, 0.3, int(np.prod(head))).astype(t), head, "b")
    y = api.tanh(api.layer_norm(api.mul(x, x), w, b, ndims=ndims, epsilon=1e-3))
    loss = api.reduce_sum(api.mul(y, api.square(y)))
    return loss, [x, w, b]


@pytest.mark.parametrize("ndims", [1, 2])
def test_graph_gradients_against_differences(ndims):
    """Central differences in double: a step of 1e-6 leaves 1e-12 (its square) and 1e-10 (the loss's
    roundings over the step) of values of the loss's size; 1e-7 of it is asked for."""
    from tenncor_amd import graph
    graph.set_evaluator("plain")
    try:
        g = graph.Graph()
        api = graph.Api(g)
        loss, leaves = layer_graph(g, api, np.float64, ndims=ndims)
        grads = g.derive(loss, leaves)
        g.evaluate([loss] + grads)
        got = [d.get() for d in grads]
        for leaf, grad in zip(leaves, got):
            base = leaf.get().copy()
            for i in np.random.default_rng(1).choice(base.size, min(base.size, 8), replace=False):
                value = []
                for step in (1e-6, -1e-6):
                    moved = base.copy()
                    moved[i] += step
                    g.assign(leaf, moved)
                    g.evaluate([loss])
                    value.append(loss.get()[0])
                assert abs((value[0] - value[1]) / 2e-6 - grad[i]) <= 1e-7 * max(1, abs(value[0]))
            g.assign(leaf, base)
        g.close()
    finally:
        graph.set_evaluator("default")


@pytest.mark.parametrize("shape,ndims", [((12, 5, 3), 1), ((40, 300), 1), ((8, 6, 70), 2)])
def test_graph_under_every_evaluator(shape, ndims):
    """The walk, recordings launch by launch (the same bits) and the default evaluator, leaves
    re-assigned between passes."""
    from tenncor_amd import graph
    seen = {}
    try:
        for kind in ("plain", "replay_launches", "replay", "replay_unfused"):
            graph.set_evaluator(kind)
            g = graph.Graph()
            api = graph.Api(g)
            loss, leaves = layer_graph(g, api, np.float32, shape=shape, ndims=ndims)
            targets = [loss] + g.derive(loss, leaves)
            seen[kind] = []
            first = leaves[0].get().copy()
            for k in range(4):
                g.assign(leaves[0], first * np.float32(1 + 0.25 * k))
                g.evaluate(targets)
                seen[kind].append([v.get().copy() for v in targets])
            if kind != "plain":
                assert graph.evaluator_stats()["record_failures"] == 0, graph.evaluator_stats()
            g.close()
    finally:
        graph.set_evaluator("default")
    for kind, rows in seen.items():
        for got, want in zip(rows, seen["plain"]):
            for a, b in zip(got, want):
                if kind in ("replay_launches", "replay_unfused"):
                    np.testing.assert_array_equal(a, b)
                else:
                    assert abs(a - b).max() <= 1e-5 * max(abs(b).max(), 1e-30)
