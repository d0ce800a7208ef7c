"""tcg_orthogonalize against the iteration in 64 bits, ORTHOGONALIZE nodes and
the update rule in graphs, and a training step with layer normalisation.

Tolerances, of the Frobenius norm of the difference.  Let X_k be the iterates in
64 bits and D the largest slope of the polynomial p (of |p'| and |p(s)| / s) over
the singular values they can have: a perturbation e of X_k is one of at most D |e|
of X_k+1 (the divided differences of p are bounded by D).  A step adds, relative
to |X_k|, the roundings of its operands -- for the halves of fp32 2^-22 each, of X
and of A and B, B's norm being at most 4 here -- and of its sums, which add up as
a random walk over at most 48 additions of 2^-24 each: together at most
8 * 2^-22.  In double an operand is rounded by 2^-53 and a sum over k indices is
off by k 2^-53 of its magnitudes at most: (8 + k) 2^-53 sqrt(m).  Summed over the
steps: tol = eta sum_k D^(steps - 1 - k) |X_k|.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

COEF = (3.4445, -4.7750, 2.0315)
CODE = {np.float32: 2, np.float64: 1}


@pytest.fixture(scope="module")
def ctx():
    from tenncor_amd import capi
    c = capi.Context(0)
    yield c
    c.close()


def reference(g, steps=5, coef=COEF, eps=1e-7):
    """The result in 64 bits and sum_k D^(steps - 1 - k) |X_k|."""
    a, b, c = coef
    x = g.astype(np.float64)
    norm = np.linalg.norm(x)
    x = x / (norm + eps) if norm + eps > 0 else x * np.nan
    tall = x.shape[0] > x.shape[1]
    if tall:
        x = x.T
    top, size = 1.0, 0.0
    slopes, norms = [], []
    for _ in range(steps):
        s = np.linspace(0, top, 4001)
        slopes.append(max(abs(a + 3 * b * s ** 2 + 5 * c * s ** 4).max(), abs(a + b * s ** 2 + c * s ** 4).max(), 1.0))
        norms.append(np.linalg.norm(x))
        gram = x @ x.T
        x = a * x + (b * gram + c * (gram @ gram)) @ x
        top = abs(s * (a + b * s ** 2 + c * s ** 4)).max() * 1.001
    for k in range(steps):
        size += np.prod(slopes[k + 1:]) * norms[k]
    return (x.T if tall else x), size


def eta(t, shape):
    low, high = min(shape), max(shape)
    return 8 * 2.0 ** -22 if t == np.float32 else (8 + high) * 2.0 ** -53 * np.sqrt(low)


def close(got, g, steps=5, coef=COEF, eps=1e-7):
    want, size = reference(g, steps, coef, eps)
    assert np.isfinite(got).all()
    off = np.linalg.norm(got.astype(np.float64) - want)
    tol = eta(g.dtype.type, g.shape) * size
    assert off <= tol, "%g of the tolerance, %g of the result" % (off / tol, off / np.linalg.norm(want))


MARK = -77.0


def run(ctx, g, pad=0, gap=0, shift=0, in_place=False, **more):
    """g: [batch][rows][cols]; pad elements between rows, gap between matrices."""
    t = g.dtype.type
    batch, rows, cols = g.shape
    ld = cols + pad
    stride = rows * ld + gap

    def lay(v):
        host = np.full(shift + batch * stride, MARK, t)
        for z in range(batch):
            host[shift + z * stride:shift + z * stride + rows * ld].reshape(rows, ld)[:, :cols] = v[z]
        return host

    src = ctx.upload(lay(g))
    dst = src if in_place else ctx.upload(lay(np.zeros_like(g)))
    size = g.itemsize * shift
    ctx.orthogonalize(CODE[t], rows, cols, batch, src.ptr + size, ld, stride, dst.ptr + size, ld, stride, **more)
    flat = dst.get()
    out = np.stack([flat[shift + z * stride:shift + z * stride + rows * ld].reshape(rows, ld)[:, :cols].copy() for z in range(batch)])
    for z in range(batch):
        flat[shift + z * stride:shift + z * stride + rows * ld].reshape(rows, ld)[:, :cols] = MARK
    assert (flat == MARK).all(), "wrote between the rows"
    if not in_place:
        np.testing.assert_array_equal(src.get(), lay(g))
    return out


def gradient(rows, cols, t=np.float32, batch=1, seed=0, scale=1e-3):
    """A few strong directions and noise."""
    rng = np.random.default_rng(seed)
    rank = min(8, rows, cols)
    out = [(rng.normal(0, 1, (rows, rank)) * np.linspace(1, 0.1, rank)) @ rng.normal(0, 1, (rank, cols)) +
           0.05 * rng.normal(0, 1, (rows, cols)) for _ in range(batch)]
    return (np.stack(out) * scale).astype(t)


SIZES = [(1, 1), (1, 9), (9, 1), (2, 3), (7, 7), (31, 33), (32, 32), (33, 31), (64, 64), (64, 65), (65, 64), (63, 130), (40, 500), (500, 40),
         (3, 1200), (96, 97), (128, 128), (128, 160), (129, 128), (130, 129), (100, 310), (257, 300), (300, 257), (200, 1000), (1000, 203),
         (513, 777), (640, 384), (4, 4096)]


@pytest.mark.parametrize("t", [np.float32, np.float64])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_one_matrix(ctx, rows, cols, t):
    g = gradient(rows, cols, t, seed=rows * 4099 + cols)
    for pad, shift in ((0, 0), (3, 1)):
        close(run(ctx, g, pad=pad, shift=shift)[0], g[0])


@pytest.mark.parametrize("t", [np.float32, np.float64])
@pytest.mark.parametrize("batch,rows,cols", [(2, 5, 9), (4, 64, 96), (7, 70, 40), (3, 129, 140), (300, 9, 17), (2, 400, 260)])
def test_several_matrices(ctx, batch, rows, cols, t):
    g = gradient(rows, cols, t, batch, seed=3)
    got = run(ctx, g, pad=2, gap=5)
    for z in range(batch):
        close(got[z], g[z])
    # a matrix by itself gives what it gives among others wherever the same tiles are used for both
    again = run(ctx, g, pad=2, gap=5)
    np.testing.assert_array_equal(got, again)


# 3, 8, 17, 2 and 5 workgroups to a tile of A on 256 CUs, mostly with a shorter last run of slabs
SHARED = [(1, 700, 2000), (1, 260, 3100), (1, 40, 9900), (3, 1000, 330), (2, 190, 2101)]


@pytest.mark.parametrize("batch,rows,cols", SHARED)
def test_tiles_that_workgroups_share(ctx, batch, rows, cols):
    g = gradient(rows, cols, batch=batch, seed=rows)
    got = run(ctx, g, pad=1, gap=3)
    for z in range(batch):
        close(got[z], g[z])
    for _ in range(10):  # whoever arrives last, the sums are the same
        np.testing.assert_array_equal(got, run(ctx, g, pad=1, gap=3))


def test_shared_tiles_recorded_and_beside_a_fork(ctx):
    g, h = gradient(260, 3100, seed=1), gradient(260, 3100, seed=2)
    wants = [run(ctx, v)[0].reshape(-1) for v in (g, h)]
    srcs = [ctx.upload(v) for v in (g, h)]
    dsts = [ctx.upload(np.zeros_like(v)) for v in (g, h)]

    def both():
        ctx.fork()
        ctx.orthogonalize(2, 260, 3100, 1, srcs[0].ptr, 3100, 0, dsts[0].ptr, 3100, 0)
        ctx.fork_end()
        ctx.orthogonalize(2, 260, 3100, 1, srcs[1].ptr, 3100, 0, dsts[1].ptr, 3100, 0)
        ctx.join()

    def check():
        for dst, want in zip(dsts, wants):
            np.testing.assert_array_equal(dst.get(), want)
            ctx.fill_zero(dst.ptr, dst.nbytes)

    both()
    check()
    ctx.capture_begin()
    both()
    graph = ctx.capture_end()
    for _ in range(3):
        ctx.graph_launch(graph)
        check()
        both()
        check()
    ctx.graph_destroy(graph)


@pytest.mark.parametrize("rows,cols", [(2000, 2050), (2100, 1900)])
def test_a_large_matrix(ctx, rows, cols):
    """Enough tiles of 128 x 128 for the chip; singular values of every size, the weakest near zero."""
    g = np.random.default_rng(2).normal(0, 1, (1, rows, cols)).astype(np.float32)
    close(run(ctx, g)[0], g[0])


@pytest.mark.parametrize("rows,cols", [(40, 56), (300, 200)])
@pytest.mark.parametrize("t", [np.float32, np.float64])
def test_steps_and_coefficients(ctx, rows, cols, t):
    from tenncor_amd import capi
    g = gradient(rows, cols, t, seed=11)
    for steps, coef in ((1, COEF), (2, COEF), (3, (1.5, -0.5, 0.0)), (8, (1.875, -1.25, 0.375)), (2, (1.0, 0.0, 0.0)), (2, (0.0, 0.0, 0.0)),
                        (4, (10.0, 0.0, 0.0)), (3, (2.0, 1.0, 0.5)), (3, (-3.0, 4.0, -1.5))):
        if coef == (2.0, 1.0, 0.5):
            # 1 -> 3.5 -> 312.5 -> 1.5e12: past the 1e6 that the documentation names
            with pytest.raises(capi.TcgError, match="grow past"):
                run(ctx, g, steps=steps, coef=coef)
            continue
        got = run(ctx, g, steps=steps, coef=coef)[0]
        close(got, g[0], steps, coef)
    # a thousandth of a matrix, a large epsilon
    close(run(ctx, g, eps=3.0)[0], g[0], eps=3.0)


def test_the_result_is_near_orthogonal(ctx):
    """What the operator is for: every singular value of the result between 0.6 and 1.25
    (the range of p after five steps for values above 1e-2 of the norm)."""
    rng = np.random.default_rng(5)
    u, _ = np.linalg.qr(rng.normal(0, 1, (90, 60)))
    v, _ = np.linalg.qr(rng.normal(0, 1, (70, 60)))
    g = ((u * np.linspace(1, 0.2, 60)) @ v.T).astype(np.float32)[None]
    s = np.linalg.svd(run(ctx, g)[0].astype(np.float64), compute_uv=False)[:60]
    assert s.min() > 0.6 and s.max() < 1.25


@pytest.mark.parametrize("rows,cols", [(20, 30), (200, 150)])
def test_a_power_of_two_changes_nothing(ctx, rows, cols):
    """G and 2^k G are the same to the bit without epsilon: the norm's square is taken in a
    type that neither overflows nor loses its small values."""
    g = gradient(rows, cols, seed=4, scale=1.0)
    want = run(ctx, g, eps=0.0)
    for k in (-100, -60, 60, 110):
        np.testing.assert_array_equal(run(ctx, np.ldexp(g, k).astype(np.float32), eps=0.0), want)


@pytest.mark.parametrize("rows,cols", [(12, 20), (150, 140)])
@pytest.mark.parametrize("t", [np.float32, np.float64])
def test_zeros_and_values_that_are_none(ctx, rows, cols, t):
    g = gradient(rows, cols, t, 4, seed=6)
    alone = run(ctx, g)
    g[1] = 0
    g[2, rows // 2, cols - 1] = np.nan
    got = run(ctx, g)
    assert not got[1].any() and np.isnan(got[2]).all()
    np.testing.assert_array_equal(got[[0, 3]], alone[[0, 3]])
    g[2, rows // 2, cols - 1] = np.inf
    got = run(ctx, g)
    assert np.isnan(got[2]).all()
    np.testing.assert_array_equal(got[[0, 3]], alone[[0, 3]])
    assert np.isnan(run(ctx, np.zeros((1, rows, cols), t), eps=0.0)).all()


@pytest.mark.parametrize("t", [np.float32, np.float64])
@pytest.mark.parametrize("rows,cols", [(30, 50), (50, 30), (260, 200)])
def test_in_place(ctx, rows, cols, t):
    g = gradient(rows, cols, t, 3, seed=8)
    np.testing.assert_array_equal(run(ctx, g, pad=1, gap=2, in_place=True), run(ctx, g, pad=1, gap=2))


def test_nothing_to_do(ctx):
    for rows, cols, batch in ((0, 4, 1), (4, 0, 1), (4, 4, 0)):
        ctx.orthogonalize(2, rows, cols, batch, None, cols, 0, None, cols, 0)


def test_refusals(ctx):
    from tenncor_amd import capi
    a, b = ctx.upload(np.zeros(64, np.float32)), ctx.upload(np.zeros(64, np.float32))

    def call(dtype=2, rows=4, cols=4, batch=2, src=a.ptr, ldi=4, stride_i=16, dst=b.ptr, ldo=4, stride_o=16, **more):
        ctx.orthogonalize(dtype, rows, cols, batch, src, ldi, stride_i, dst, ldo, stride_o, **more)

    for args, match in [({"dtype": 3}, "neither float nor double"), ({"ldi": 3}, "leading dims"), ({"ldo": 3}, "leading dims"),
                        ({"steps": 0}, "steps"), ({"steps": 65}, "steps"), ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"),
                        ({"src": None}, "NULL"), ({"dst": None}, "NULL"), ({"stride_i": 15}, "overlap"), ({"stride_o": 15}, "overlap"),
                        ({"dst": a.ptr, "ldo": 5, "stride_o": 20}, "in place"), ({"rows": 1 << 40, "stride_i": 1 << 50, "stride_o": 1 << 50}, "too large"),
                        ({"batch": 1 << 20}, "too many"), ({"coef": (10.0, 0.0, 0.0), "steps": 20}, "grow"),
                        ({"coef": (float("nan"), 0.0, 0.0)}, "grow"), ({"coef": (1.0, float("inf"), 0.0)}, "grow")]:
        with pytest.raises(capi.TcgError, match=match):
            call(**args)
    ctx.sync()
    assert not a.get().any() and not b.get().any()
    ctx.capture_begin(small=True)
    with pytest.raises(capi.TcgError) as err:
        call()
    assert err.value.status == 3
    ctx.capture_abort()


def test_recorded_and_replayed(ctx):
    """Two recordings with workspaces of their own, replayed in turn between eager calls."""
    cases = []
    for shape, t in (((1, 40, 60), np.float32), ((1, 300, 200), np.float32), ((2, 70, 50), np.float64)):
        g = gradient(shape[1], shape[2], t, shape[0], seed=9)
        src, dst = ctx.upload(g), ctx.upload(np.zeros_like(g))
        n, code = g.size, CODE[t]

        def call(src=src, dst=dst, shape=shape, code=code):
            batch, rows, cols = shape
            ctx.orthogonalize(code, rows, cols, batch, src.ptr, cols, rows * cols, dst.ptr, cols, rows * cols)

        call()
        want = dst.get()
        ctx.capture_begin()
        call()
        cases.append((ctx.capture_end(), src, dst, want, call, n, code))
    for _ in range(3):
        for _, src, dst, want, call, n, code in cases:
            ctx.ew_unary("SQUARE", code, n, src.ptr, dst.ptr)
            ctx.d2d(dst.ptr, src.ptr, dst.nbytes)
            call()
            ctx.sync()
            ctx.fill_zero(dst.ptr, dst.nbytes)
        for graph, *_ in cases:
            ctx.graph_launch(graph)
        for _, src, dst, want, *_ in cases:
            np.testing.assert_array_equal(dst.get(), want)
    for graph, *_ in cases:
        ctx.graph_destroy(graph)


def test_beside_a_fork_and_in_a_batch(ctx):
    g = gradient(150, 130, seed=10)
    want = run(ctx, g)[0].reshape(-1)
    src, one, two, neg = (ctx.upload(v) for v in (g, np.zeros_like(g), np.zeros_like(g), np.zeros_like(g)))
    ctx.fork()
    ctx.orthogonalize(2, 150, 130, 1, src.ptr, 130, 0, one.ptr, 130, 0)
    ctx.fork_end()
    ctx.orthogonalize(2, 150, 130, 1, src.ptr, 130, 0, two.ptr, 130, 0)
    ctx.join()
    np.testing.assert_array_equal(one.get(), want)
    np.testing.assert_array_equal(two.get(), want)
    small = gradient(9, 11, seed=10)
    src = ctx.upload(small)
    ctx.batch_begin()
    ctx.ew_unary("NEG", 2, 99, src.ptr, neg.ptr)
    ctx.orthogonalize(2, 9, 11, 1, neg.ptr, 11, 0, one.ptr, 11, 0)
    ctx.batch_end()
    np.testing.assert_array_equal(one.get()[:99], run(ctx, -small)[0].reshape(-1))


def test_memory_goes_back(ctx):
    before, _ = ctx.mem_stats()
    g = gradient(200, 300, seed=1)
    run(ctx, g)
    assert ctx.mem_stats()[0] <= before + 4096 * 1024  # buffers of this test's own, if not collected yet
    src, dst = ctx.upload(g), ctx.empty(g.size, np.float32)
    held, _ = ctx.mem_stats()
    for _ in range(5):
        ctx.orthogonalize(2, 200, 300, 1, src.ptr, 300, 0, dst.ptr, 300, 0)
    assert ctx.mem_stats()[0] == held


def test_ops(ctx):
    from tenncor_amd import ops
    g = gradient(12, 20, batch=6, seed=12)
    got = ops.orthogonalize(ops.from_host(ctx, g, [20, 12, 3, 2])).get().reshape(6, 12, 20)
    for z in range(6):
        close(got[z], g[z])


# ---- in graphs ------------------------------------------------------------------

def training(g, t, seed=0, batch=24, nin=20, hid=36, nout=6, rate=0.05):
    """dense -> layer norm -> tanh -> dense, squared error; the matrices by muon, the
    layer norm's weight and bias by sgd."""
    from tenncor_amd import graph
    api, rng = graph.Api(g), np.random.default_rng(seed)
    values = {"x": rng.normal(0, 1, (batch, nin)), "y": rng.normal(0, 1, (batch, nout)), "w0": rng.normal(0, 0.3, (nin, hid)),
              "w1": rng.normal(0, 0.3, (hid, nout)), "w": rng.normal(1, 0.1, hid), "b": rng.normal(0, 0.1, hid)}
    v = {k: g.variable(u.astype(t), list(u.shape[::-1]), k) for k, u in values.items()}
    h = api.tanh(api.layer_norm(api.matmul(v["x"], v["w0"]), v["w"], v["b"]))
    out = api.matmul(h, v["w1"])
    loss = api.reduce_mean(api.square(api.sub(out, v["y"])))
    approx = graph.Approx(api)
    updates = approx.muon(loss, [v["w0"], v["w1"]], learning_rate=rate) + approx.sgd(loss, [v["w"], v["b"]], learning_rate=rate)
    return loss, v, updates, approx, {k: u.astype(t).astype(np.float64) for k, u in values.items()}


def training_by_hand(p, steps, rate=0.05, decay=0.95, eps=1e-5):
    """The same in 64 bits.  Updates are assignments in the order they are listed, and each
    rule has a gradient graph of its own: sgd's gradients, behind muon's assignments, read
    the second matrix as those left it."""
    p, m, losses = dict(p), {"w0": 0.0, "w1": 0.0}, []
    for _ in range(steps):
        z = p["x"] @ p["w0"]
        mean = z.mean(1, keepdims=True)
        r = 1 / np.sqrt(((z - mean) ** 2).mean(1, keepdims=True) + eps)
        xh = (z - mean) * r
        h = np.tanh(xh * p["w"] + p["b"])
        d = h @ p["w1"] - p["y"]
        losses.append((d ** 2).mean())
        do = 2 * d / d.size
        dn = (do @ p["w1"].T) * (1 - h ** 2)
        gw = dn * p["w"]
        dz = r * (gw - gw.mean(1, keepdims=True) - xh * (gw * xh).mean(1, keepdims=True))
        grads = {"w0": p["x"].T @ dz, "w1": h.T @ do}
        for k in ("w0", "w1"):
            m[k] = decay * m[k] + grads[k]
            step, _ = reference(grads[k] + decay * m[k])
            p[k] = p[k] - rate * max(1, p[k].shape[0] / p[k].shape[1]) ** 0.5 * step
        dn = (do @ p["w1"].T) * (1 - h ** 2)
        p["w"] = p["w"] - rate * (dn * xh).sum(0)
        p["b"] = p["b"] - rate * dn.sum(0)
    return p, losses


@pytest.mark.parametrize("t", [np.float32, np.float64])
def test_training_steps_under_every_evaluator(t):
    """Four steps of the whole: in double against the same by hand (1e-9: a step's own error is
    1e-13, which the iteration's slope takes to 485 of it a step, and tanh's gradient passes on),
    and the recorded passes against the walk, bit for bit launch by launch."""
    from tenncor_amd import graph
    steps, seen = 4, {}
    try:
        for kind in ("plain", "replay_launches", "replay", "replay_unfused"):
            graph.set_evaluator(kind)
            g = graph.Graph()
            loss, v, updates, approx, start = training(g, t)
            step = approx.apply_update(loss, updates)
            losses = []
            for _ in range(steps):
                g.evaluate([step])
                losses.append(step.get()[0])
            seen[kind] = [np.array(losses)] + [v[k].get().copy() for k in ("w0", "w1", "w", "b")]
            if kind != "plain":
                assert graph.evaluator_stats()["record_failures"] == 0, graph.evaluator_stats()
            g.close()
    finally:
        graph.set_evaluator("default")
    want, losses = training_by_hand(start, steps)
    tol = 1e-9 if t == np.float64 else 2e-3
    for kind, got in seen.items():
        for a, b in zip(got, [np.array(losses)] + [want[k].reshape(-1) for k in ("w0", "w1", "w", "b")]):
            assert abs(a - b).max() <= tol * max(1, abs(b).max()), kind
        if kind in ("replay_launches", "replay_unfused"):
            for a, b in zip(got, seen["plain"]):
                np.testing.assert_array_equal(a, b)
