"""More rows than one sweep of the grid, in every shape of the kernels.  Tolerances as in
test_gpu_layer_norm; where a sum over rows runs longer than there, said at the case.
"""
import numpy as np
import pytest

from test_gpu_layer_norm import close, ctx, data, reference, run_backward, run_forward  # noqa: F401 (ctx is a fixture)

pytestmark = pytest.mark.gpu


# 16, 32 and 64 lanes a row (8192 workgroups of 16, 8 and 4 rows), 256 and 1024 (of one row)
@pytest.mark.parametrize("rows,cols", [(140000, 60), (70000, 100), (40000, 500), (9000, 1100), (9001, 2050), (8500, 4100), (8193, 8200)])
def test_forward(ctx, rows, cols):
    t = np.float32
    x, w, b, _ = data(rows, cols, t, rows)
    y, mean, rstd = run_forward(ctx, x, w, b, 1e-5, pad=1)
    want = reference(x, w, b, 1e-5)
    close(y, want["y"], want["y_size"], 160, t)
    close(mean, want["mean"], abs(want["mean"]) + 90 / want["rstd"], 2, t)
    close(rstd, want["rstd"], want["rstd"], 50, t)


@pytest.mark.parametrize("rows,cols", [(9000, 300), (8200, 1030)])
def test_forward_in_double(ctx, rows, cols):
    t = np.float64
    x, w, b, _ = data(rows, cols, t, rows)
    y, _, _ = run_forward(ctx, x, w, b, 1e-5)
    want = reference(x, w, b, 1e-5)
    close(y, want["y"], want["y_size"], 160, t)


@pytest.mark.parametrize("rows,cols,t", [(2100, 33000, np.float32), (1030, 33000, np.float64)])
def test_rows_beyond_registers(ctx, rows, cols, t):
    """Over 8192 chunks, and over 1024 rows, whose sums are 64 additions long at most and
    then one for each of 16 to 32 parts."""
    x, w, b, g = data(rows, cols, t, rows)
    want = reference(x, w, b, 1e-5, g)
    y, _, _ = run_forward(ctx, x, w, b, 1e-5)
    close(y, want["y"], want["y_size"], 160, t)
    del y
    got = run_backward(ctx, g, x, w, 1e-5)
    close(got["dx"], want["dx"], want["dx_size"], 300, t)
    close(got["dw"], want["dw"], want["dw_size"], 300, t)
    close(got["db"], want["db"], want["db_size"], 150, t)


def test_more_rows_beyond_registers_than_parts_of_64(ctx):
    """8200 rows (820 ten times), 128 parts: 65 additions and 127, each of 2^-24 of a partial sum at
    most: 200 for db, and the 150 of h and two roundings besides for dw."""
    t = np.float32
    x, w, b, g = data(820, 16385, t, 1)
    want = reference(x, w, b, 1e-5, g)
    got = run_backward(ctx, np.tile(g, (10, 1)), np.tile(x, (10, 1)), w, 1e-5, want=("dw", "db"))
    close(got["dw"], 10 * want["dw"], 10 * want["dw_size"], 352, t)
    close(got["db"], 10 * want["db"], 10 * want["db_size"], 200, t)


def test_a_row_of_more_than_2_to_31_elements(ctx):
    """A pattern of 100003 elements over and over; looked at where it begins, around 2^31 and 2^32
    bytes, around 2^31 elements and where it ends.  With dy = x and epsilon 1, h = (x - m) r:
    dx = r (x - m - h mean(x h)), mean(x h) = (1 - r^2) / r, dw = x h.  Statistics meet in double."""
    t, period, cols = np.float32, 100003, (1 << 31) + 70001
    p = np.random.default_rng(3).normal(0.5, 1, period).astype(t)
    x, out, dw = (ctx.alloc(4 * cols) for _ in range(3))
    try:
        ctx.h2d(x, p)
        done = period
        while done < cols:  # whole periods double
            n = min(done, cols - done)
            ctx.d2d(x + 4 * done, x, 4 * n)
            done += n
        wide = p.astype(np.float64)
        whole, rest = cols // period, cols % period
        m = (whole * wide.sum() + wide[:rest].sum()) / cols
        d = wide - m
        r = 1 / np.sqrt((whole * (d ** 2).sum() + (d[:rest] ** 2).sum()) / cols + 1)
        h = d * r
        places = [0, (1 << 29) - 3000, (1 << 30) - 3000, (1 << 31) - 3000, cols - 5000]

        def check(ptr, want, size, steps):
            for at in places:
                got = ctx.d2h(ptr + 4 * at, 5000, t)
                i = np.arange(at, at + 5000) % period
                close(got, want[i], size[i], steps, t)

        ctx.layer_norm(2, 1, cols, x, cols, None, None, 1.0, out, cols)
        check(out, h, abs(h) + 1, 160)
        ctx.layer_norm_grad(2, 1, cols, x, cols, x, cols, None, 1.0, dx=out, lddx=cols, dweight=dw)
        along = (1 - r * r) / r
        big = abs(h) + 1
        check(out, r * (d - h * along), r * (abs(wide) + abs(wide).mean() + big * abs(wide).mean() + big * (abs(wide) * big).mean()), 300)
        check(dw, wide * h, abs(wide) * big, 300)
    finally:
        for buf in (x, out, dw):
            ctx.free(buf, 4 * cols)
