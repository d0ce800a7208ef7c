"""ORTHOGONALIZE nodes and the update rule built on them, without a GPU."""
import numpy as np
import pytest


@pytest.fixture()
def g():
    from tenncor_amd import graph
    gr = graph.Graph()
    yield gr
    gr.close()


@pytest.fixture()
def api(g):
    from tenncor_amd import graph
    return graph.Api(g)


def var(g, shape, dtype=np.float32, label="x"):
    return g.variable(np.arange(int(np.prod(shape)), dtype=dtype), shape, label)


@pytest.mark.parametrize("shape", [[1], [5], [4, 3], [3, 4, 2], [3, 4, 2, 2]])
def test_the_result_has_the_shape_of_its_operand(g, api, shape):
    out = api.orthogonalize(var(g, shape), steps=3, epsilon=0.5, coef=(1.5, -0.5, 0.0))
    assert out.shape == shape + [1] * (8 - len(shape))
    assert g.attr(out, "reals") == [3.0, 0.5, 1.5, -0.5, 0.0]
    assert g.launch_plan([out])[0] == "node ORTHOGONALIZE"


@pytest.mark.parametrize("reals,match", [
    ([5, 1e-7, 1, 1], "three coefficients"), ([0, 0, 1, 1, 1], "steps"), ([65, 0, 1, 1, 1], "steps"), ([2.5, 0, 1, 1, 1], "steps"),
    ([float("nan"), 0, 1, 1, 1], "steps"), ([5, -1, 1, 1, 1], "epsilon"), ([5, float("nan"), 1, 1, 1], "epsilon")])
def test_parameters_that_make_no_sense_are_refused(g, reals, match):
    from tenncor_amd import graph
    with pytest.raises(graph.GraphError, match=match):
        g.functor("ORTHOGONALIZE", [var(g, [4, 3])], reals=reals)


def test_operands_that_do_not_fit_are_refused(g, api):
    from tenncor_amd import graph
    with pytest.raises(graph.GraphError, match="integers"):
        api.orthogonalize(var(g, [4, 3], np.int32))
    x = var(g, [4, 3])
    with pytest.raises(graph.GraphError, match="2 arguments"):
        g.functor("ORTHOGONALIZE", [x, x], reals=[5, 0, 1, 1, 1])
    out = api.orthogonalize(x)
    with pytest.raises(graph.GraphError, match="cannot derive ORTHOGONALIZE"):
        g.local_derivative(out, x, 0)


def test_the_update_rule_is_a_graph_like_the_others(g, api):
    from tenncor_amd import graph
    x, w = var(g, [4, 3]), var(g, [6, 4])
    loss = api.reduce_sum(api.square(api.matmul(x, w)))
    approx = graph.Approx(api)
    ((target, step),) = approx.muon(loss, [w])
    assert target.id == w.id and g.opcode(step) == "ASSIGN_SUB"
    assert [v.shape for v in approx.slots["momentum"]] == [w.shape]
    text = g.to_string(step)
    assert text.count("(ORTHOGONALIZE") == 1 and "(ASSIGN<" in text or "(ASSIGN" in text
    with pytest.raises(ValueError, match="matrices"):
        graph.Approx(api).muon(loss, [var(g, [3, 4, 2])])


def test_three_coefficients():
    from tenncor_amd import capi
    for coef in ((1.5, -0.5), (1, 2, 3, 4)):
        with pytest.raises(ValueError, match="not %d of them" % len(coef)):
            capi.Context.orthogonalize(None, 2, 1, 1, 1, 0, 1, 1, 0, 1, 1, coef=coef)
