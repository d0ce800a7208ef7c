"""The step length of the update rule ``muon``: the published factor is the root of
max(1, fan-out / fan-in) of a layer's weights, which here are {outputs, inputs}
(dim 0 counts outputs: matmul(x, w) and dense sum over dim 1 of w).
"""
import numpy as np
import pytest

from test_gpu_orthogonalize import close, reference, training

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("inputs,outputs", [(12, 48), (48, 12), (30, 30), (9, 1), (2, 9)])
@pytest.mark.parametrize("layer", ["matmul", "dense"])
def test_a_layer_moves_by_its_fan(inputs, outputs, layer):
    """One update without momentum: (old - new) / rate / sqrt(max(1, outputs / inputs)) is the
    orthogonalised gradient.  Weights of zero, so that their update is kept to its last bit."""
    from tenncor_amd import graph
    rng = np.random.default_rng(inputs)
    x = rng.normal(0, 1, (20, inputs))
    up = rng.normal(0, 1, (20, outputs))
    g = graph.Graph()
    api = graph.Api(g)
    vx = g.variable(x.reshape(-1), [inputs, 20], "x")
    w = g.variable(np.zeros(inputs * outputs), [outputs, inputs], "w")
    y = api.matmul(vx, w) if layer == "matmul" else api.dense(vx, w)
    loss = api.reduce_sum(api.mul(y, g.variable(up.reshape(-1), [outputs, 20], "up")))
    approx = graph.Approx(api)
    step = approx.apply_update(loss, approx.muon(loss, [w], learning_rate=0.5, decay=0.0))
    g.evaluate([step])
    moved = -w.get().reshape(inputs, outputs) / (0.5 * max(1.0, outputs / inputs) ** 0.5)
    g.close()
    close(moved, x.T @ up)


def by_hand(p, steps, rate=0.05, decay=0.95, eps=1e-5):
    """The training of test_gpu_orthogonalize in 64 bits, the matrices' steps by outputs over inputs."""
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
        for k, grad in (("w0", p["x"].T @ dz), ("w1", h.T @ do)):
            m[k] = decay * m[k] + grad
            inputs, outputs = p[k].shape
            p[k] = p[k] - rate * max(1.0, outputs / inputs) ** 0.5 * reference(grad + decay * m[k])[0]
        # the layer normalisation's updates come behind the matrices' and read the second one as it is then
        dn = (do @ p["w1"].T) * (1 - h ** 2)
        p["w"], p["b"] = p["w"] - rate * (dn * xh).sum(0), p["b"] - rate * dn.sum(0)
    return p, losses


@pytest.mark.parametrize("t", [np.float32, np.float64])
def test_training_steps_under_every_evaluator(t):
    """Four steps of dense -> layer norm -> tanh -> dense, the matrices by muon (20 to 36 and 36 to 6
    units), against the same by hand: 1e-9 in double (a step's own error is 1e-13, which the
    iteration's slope takes to 485 of it a step, and tanh's gradient passes on), 2e-3 in float for
    the same reason; recordings launch by launch give the walk's bits."""
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
    want, losses = by_hand(start, steps)
    tol = 1e-9 if t == np.float64 else 2e-3
    for kind, got in seen.items():
        for a, b in zip(got, [np.array(losses)] + [want[k].reshape(-1) for k in ("w0", "w1", "w", "b")]):
            assert abs(a - b).max() <= tol * max(1, abs(b).max()), kind
        if kind in ("replay_launches", "replay_unfused"):
            for a, b in zip(got, seen["plain"]):
                np.testing.assert_array_equal(a, b)
