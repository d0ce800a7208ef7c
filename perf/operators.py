"""The operators of training that this package offers beside the nodes of the
reference's graphs, as workloads: layer normalisation (forward, and the three
gradients) and the orthogonalised update of a weight matrix by a polynomial
iteration of matrix products.

Matrices are row-major: `rows` rows of `cols` elements, which as a tenncor
shape is {cols, rows} (dim 0 fastest).  With `own` false the functions compute
the operators in elementary torch operations, with `own` true through
``tenncor_amd.capi``.
"""
import math

import torch

own = False

EPSILON = 1e-5          # added to a row's variance
NORM_EPSILON = 1e-7     # added to a matrix's norm
COEF = (3.4445, -4.7750, 2.0315)
STEPS = 5

TYPES = {"float": torch.float32, "double": torch.float64}
DTYPE_CODE = {"float": 2, "double": 1}  # enum tcg_dtype

# the largest listed cases, which no drawn case exceeds
MOST_ELEMENTS = 32768 * 4096
MOST_PRODUCT = 4096 ** 3


def listed():
    return [
        # four sequences decoded one step at a time through a layer of 512 hidden units
        {"name": "norm step", "op": "norm", "type": "float", "rows": 4, "cols": 512, "pad": 0, "bias": True},
        # every hidden output of a recurrent layer: 64 steps of a batch of 256, 512 units
        {"name": "norm sequence", "op": "norm", "type": "float", "rows": 16384, "cols": 512, "pad": 0, "bias": True},
        # odd extents, rows a few elements apart from each other (a slice of a wider tensor), no bias
        {"name": "norm ragged", "op": "norm", "type": "float", "rows": 4099, "cols": 1537, "pad": 6, "bias": False},
        # the gradients of one time step of a batch of 256
        {"name": "norm grad step", "op": "norm grad", "type": "float", "rows": 256, "cols": 512, "pad": 0, "bias": True},
        # wide activations of a long batch: what the memory of the card has to carry
        {"name": "norm grad wide", "op": "norm grad", "type": "float", "rows": 32768, "cols": 4096, "pad": 0, "bias": True},
        # odd extents and rows apart from each other
        {"name": "norm grad ragged", "op": "norm grad", "type": "float", "rows": 2999, "cols": 777, "pad": 3, "bias": True},
        # gradients in double, as a check of a model is run
        {"name": "norm grad double", "op": "norm grad", "type": "double", "rows": 8192, "cols": 1000, "pad": 0, "bias": True},
        # the four gate matrices of a small recurrent cell, one update
        {"name": "orthogonal small", "op": "orthogonal", "type": "float", "batch": 4, "rows": 64, "cols": 96, "pad": 0},
        # the fused gate matrix of a recurrent layer of 512 units over 256 inputs
        {"name": "orthogonal gates", "op": "orthogonal", "type": "float", "batch": 1, "rows": 768, "cols": 2048, "pad": 0},
        # a tall matrix with odd extents, a column block of a wider one
        {"name": "orthogonal ragged", "op": "orthogonal", "type": "float", "batch": 2, "rows": 1111, "cols": 517, "pad": 5},
        # a large square matrix
        {"name": "orthogonal large", "op": "orthogonal", "type": "float", "batch": 1, "rows": 4096, "cols": 4096, "pad": 0},
        # a dense layer's matrix in double
        {"name": "orthogonal double", "op": "orthogonal", "type": "double", "batch": 1, "rows": 384, "cols": 640, "pad": 0},
    ]


def _spread(rng, low, high):
    """A whole number between the two, even in its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm grad", "orthogonal"])
    kind = rng.choice(["float", "float", "float", "double"])
    pad = rng.choice([0, 0, rng.randint(1, 16)])
    if op == "orthogonal":
        most = MOST_PRODUCT if kind == "float" else MOST_PRODUCT // 64
        while True:
            case = {"op": op, "type": kind, "batch": rng.choice([1, 1, rng.randint(2, 8)]),
                    "rows": _spread(rng, 4, 4096), "cols": _spread(rng, 4, 4096), "pad": pad}
            if case["batch"] * case["rows"] * case["cols"] * min(case["rows"], case["cols"]) <= most:
                return case
    most = MOST_ELEMENTS if kind == "float" else MOST_ELEMENTS // 2
    while True:
        case = {"op": op, "type": kind, "rows": _spread(rng, 1, 65536), "cols": _spread(rng, 8, 16384), "pad": pad,
                "bias": rng.random() < 0.75}
        if case["rows"] * (case["cols"] + pad) <= most:
            return case


def _rows_apart(full, cols):
    """The leading `cols` elements of every row of `full`."""
    return full[..., :cols]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    t = TYPES[case["type"]]
    rows, cols, ld = case["rows"], case["cols"], case["cols"] + case["pad"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=t)

    state = {"case": dict(case), "ld": ld}
    if case["op"] == "orthogonal":
        batch = case["batch"]
        # a gradient: a few strong directions and what is left of the batch's noise
        rank = min(16, rows, cols)
        g = 0.05 * normal(batch, rows, ld)
        for b in range(batch):
            g[b] += (normal(rows, rank) * torch.linspace(1.0, 0.1, rank, device=dev, dtype=t)) @ normal(rank, ld)
        g *= 1e-3
        state["g"] = g
        state["out"] = torch.zeros(batch, rows, cols, device=dev, dtype=t)
        return state
    # activations: rows of differing scale and offset
    scale = 0.5 + torch.rand(rows, 1, generator=gen, device=dev, dtype=t)
    state["x"] = normal(rows, ld) * scale + 0.5 * normal(rows, 1)
    state["weight"] = 1.0 + 0.1 * normal(cols)
    state["bias"] = 0.1 * normal(cols) if case["bias"] else None
    if case["op"] == "norm":
        state["y"] = torch.empty(rows, cols, device=dev, dtype=t)
        state["mean"] = torch.empty(rows, device=dev, dtype=t)
        state["rstd"] = torch.empty(rows, device=dev, dtype=t)
        return state
    state["dy"] = normal(rows, cols)
    # what the forward pass has left
    mean, rstd = [], []
    for part in _rows_apart(state["x"], cols).split(max(1, (1 << 26) // cols)):
        wide = part.double()
        m = wide.mean(1)
        mean.append(m.to(t))
        rstd.append((wide.sub(m[:, None]).square().mean(1) + EPSILON).rsqrt().to(t))
    state["mean"], state["rstd"] = torch.cat(mean), torch.cat(rstd)
    state["dx"] = torch.empty(rows, cols, device=dev, dtype=t)
    state["dweight"] = torch.empty(cols, device=dev, dtype=t)
    state["dbias"] = torch.empty(cols, device=dev, dtype=t) if case["bias"] else None
    return state


# ---- the plain forms ---------------------------------------------------------

def _norm_plain(s):
    x = _rows_apart(s["x"], s["case"]["cols"])
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = (d.square().mean(1, keepdim=True) + EPSILON).rsqrt()
    y = d * rstd * s["weight"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return {"y": y, "mean": mean[:, 0], "rstd": rstd[:, 0]}


def _norm_grad_plain(s):
    x, dy = _rows_apart(s["x"], s["case"]["cols"]), s["dy"]
    rstd = s["rstd"][:, None]
    xhat = (x - s["mean"][:, None]) * rstd
    gw = dy * s["weight"]
    dx = rstd * (gw - gw.mean(1, keepdim=True) - xhat * (gw * xhat).mean(1, keepdim=True))
    out = {"dx": dx, "dweight": (dy * xhat).sum(0)}
    if s["dbias"] is not None:
        out["dbias"] = dy.sum(0)
    return out


def _orthogonal_plain(s):
    case = s["case"]
    g = _rows_apart(s["g"], case["cols"])
    # a sum over every element, in 64 bits: a relative error of it moves every singular value alike
    norm = g.double().square().sum((1, 2), keepdim=True).sqrt().add(NORM_EPSILON).to(g.dtype)
    x = g / norm
    tall = case["rows"] > case["cols"]
    if tall:
        x = x.transpose(1, 2).contiguous()
    if case["batch"] == 1:
        x = x[0]
    a, b, c = COEF
    for _ in range(STEPS):
        gram = x @ x.transpose(-1, -2)
        factor = b * gram + c * (gram @ gram)
        # this product in 64 bits: what its sums round away grows by COEF[0] a
        # step along the weak directions, 3e-5 of the result at 4096 rows in 32 bits
        x = a * x + (factor.double() @ x.double()).to(x.dtype)
    if case["batch"] == 1:
        x = x[None]
    return x.transpose(1, 2).contiguous() if tall else x


# ---- through the framework ---------------------------------------------------

_contexts = {}


def _context():
    """One context of the library per device, kept as a program keeps it."""
    from tenncor_amd import capi
    device = torch.cuda.current_device()
    if device not in _contexts:
        _contexts[device] = capi.Context(device)
    return _contexts[device]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _run_own(s):
    case, ctx = s["case"], _context()
    rows, cols, code = case["rows"], case["cols"], DTYPE_CODE[case["type"]]
    if case["op"] == "norm":
        ctx.layer_norm(code, rows, cols, _ptr(s["x"]), s["ld"], _ptr(s["weight"]), _ptr(s["bias"]), EPSILON,
                       _ptr(s["y"]), cols, mean=_ptr(s["mean"]), rstd=_ptr(s["rstd"]))
        return {"y": s["y"], "mean": s["mean"], "rstd": s["rstd"]}
    if case["op"] == "norm grad":
        ctx.layer_norm_grad(code, rows, cols, _ptr(s["dy"]), cols, _ptr(s["x"]), s["ld"], _ptr(s["weight"]), EPSILON,
                            dx=_ptr(s["dx"]), lddx=cols, dweight=_ptr(s["dweight"]), dbias=_ptr(s["dbias"]),
                            mean=_ptr(s["mean"]), rstd=_ptr(s["rstd"]))
        out = {"dx": s["dx"], "dweight": s["dweight"]}
        if s["dbias"] is not None:
            out["dbias"] = s["dbias"]
        return out
    ctx.orthogonalize(code, rows, cols, case["batch"], _ptr(s["g"]), s["ld"], rows * s["ld"],
                      _ptr(s["out"]), cols, rows * cols, steps=STEPS, coef=COEF, eps=NORM_EPSILON)
    return s["out"]


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "norm":
        return _norm_plain(state)
    return _norm_grad_plain(state) if op == "norm grad" else _orthogonal_plain(state)


# ---- what a pass cannot do without -------------------------------------------

def work(case):
    size = 4 if case["type"] == "float" else 8
    rows, cols = case["rows"], case["cols"]
    n = rows * cols
    affine = cols * (2 if case["bias"] else 1) if case["op"] != "orthogonal" else 0
    if case["op"] == "norm":
        # x in, y out; weight, bias; the two statistics of every row
        return {"bytes": size * (2 * n + affine + 2 * rows), "flops": 8 * n}
    if case["op"] == "norm grad":
        # x and dy in, dx out; the weight in, its gradients out; the statistics in
        return {"bytes": size * (3 * n + cols + affine + 2 * rows), "flops": 14 * n}
    # a step: the Gram matrix and its square (one triangle of each, they are
    # symmetric), and the product with the iterate
    low, high = min(rows, cols), max(rows, cols)
    step = low * low * high + low ** 3 + 2 * low * low * high
    return {"bytes": size * 2 * case["batch"] * n, "flops": case["batch"] * STEPS * step}


# ---- the definitions in 64 bits ----------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "orthogonal":
        out = []
        for g in s["g"]:
            x = g[:, :case["cols"]].double()
            x = x / (torch.linalg.vector_norm(x) + NORM_EPSILON)
            tall = x.shape[0] > x.shape[1]
            for _ in range(STEPS):
                # the odd polynomial of the singular values, one power of the
                # Gram matrix after the other on the iterate itself
                if tall:
                    gram = torch.mm(x.t(), x)
                    third = torch.mm(x, gram)
                    fifth = torch.mm(third, gram)
                else:
                    gram = torch.mm(x, x.t())
                    third = torch.mm(gram, x)
                    fifth = torch.mm(gram, third)
                x = x.mul(COEF[0]).add_(third, alpha=COEF[1]).add_(fifth, alpha=COEF[2])
            out.append(x)
        return torch.stack(out)
    cols = case["cols"]
    weight = s["weight"].double()
    step = max(1, (1 << 25) // cols)
    if case["op"] == "norm":
        got = {"y": [], "mean": [], "rstd": []}
        for part in s["x"].split(step):
            wide = part[:, :cols].double()
            var, mean = torch.var_mean(wide, 1, correction=0)
            rstd = 1.0 / torch.sqrt(var + EPSILON)
            y = torch.einsum("rc,r,c->rc", wide - mean[:, None], rstd, weight)
            got["y"].append(y if s["bias"] is None else y + s["bias"].double())
            got["mean"].append(mean)
            got["rstd"].append(rstd)
        return {k: torch.cat(v) for k, v in got.items()}
    dx, dweight, dbias = [], torch.zeros_like(weight), torch.zeros_like(weight)
    for x, dy, mean, rstd in zip(*(s[k].split(step) for k in ("x", "dy", "mean", "rstd"))):
        dy, rstd = dy.double(), rstd.double()
        xhat = (x[:, :cols].double() - mean.double()[:, None]) * rstd[:, None]
        gw = dy * weight
        along = torch.stack([gw.sum(1), (gw * xhat).sum(1)], 1) / cols
        dx.append((gw - along[:, :1] - xhat * along[:, 1:]) * rstd[:, None])
        dweight += (dy * xhat).sum(0)
        dbias += dy.sum(0)
    out = {"dx": torch.cat(dx), "dweight": dweight}
    if s["dbias"] is not None:
        out["dbias"] = dbias
    return out
