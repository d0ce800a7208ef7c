"""What the update rule ``muon`` takes, without a GPU."""
import numpy as np
import pytest


@pytest.mark.parametrize("shape", [[6], [6, 1], [1], [3, 4, 2], [3, 1, 2]])
def test_variables_that_are_no_matrices_are_refused(shape):
    """A vector's orthogonalised update would be its direction, whatever its size."""
    from tenncor_amd import graph
    g = graph.Graph()
    api = graph.Api(g)
    x = g.variable(np.ones(int(np.prod(shape)), np.float32), shape, "x")
    w = g.variable(np.ones(12, np.float32), [4, 3], "w")
    loss = api.add(api.reduce_sum(api.square(x)), api.reduce_sum(api.square(w)))
    approx = graph.Approx(api)
    with pytest.raises(ValueError, match="matrices"):
        approx.muon(loss, [w, x])
    assert not approx.slots, "made a momentum before the refusal"
    g.close()


@pytest.mark.parametrize("shape", [[4, 3], [3, 4], [1, 5], [2, 2]])
def test_matrices_are_taken(shape):
    """A layer of one output among them."""
    from tenncor_amd import graph
    g = graph.Graph()
    api = graph.Api(g)
    w = g.variable(np.ones(int(np.prod(shape)), np.float32), shape, "w")
    ((target, step),) = graph.Approx(api).muon(api.reduce_sum(api.square(w)), [w])
    assert target.id == w.id and g.opcode(step) == "ASSIGN_SUB"
    g.close()
