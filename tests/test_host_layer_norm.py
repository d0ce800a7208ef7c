"""LAYER_NORM nodes without a GPU: shapes, refusals, the gradient graphs, the
launch plan, what the clean-up merges, and the argument checks of ``ops``."""
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


@pytest.mark.parametrize("shape,ndims", [([5], 1), ([5, 3], 1), ([5, 3, 2], 2), ([5, 1, 7, 2], 1), ([2] * 8, 7)])
def test_the_result_has_the_shape_of_x(g, api, shape, ndims):
    x, w, b = var(g, shape), var(g, shape[:ndims]), var(g, shape[:ndims])
    full = shape + [1] * (8 - len(shape))
    for args in ((), (w,), (w, b)):
        out = api.layer_norm(x, *args, ndims=ndims, epsilon=0.25)
        assert out.shape == full
        assert g.attr(out, "rank") == [ndims]
        assert g.attr(out, "reals") == [0.25]
    dx = g.functor("LAYER_NORM_DX", [x, x, w], rank=ndims, reals=[0.])
    dw = g.functor("LAYER_NORM_DWEIGHT", [x, x], rank=ndims, reals=[0.])
    assert dx.shape == full and dw.shape == shape[:ndims] + [1] * (8 - ndims)


def test_a_bias_without_a_weight_is_an_addition(g, api):
    x, b = var(g, [4, 3]), var(g, [4])
    out = api.layer_norm(x, bias=b)
    assert g.opcode(out) == "ADD" and sorted(g.opcode(a) for a in g.args(out)) == ["EXTEND", "LAYER_NORM"]


@pytest.mark.parametrize("rank,reals,match", [
    (0, [1e-5], "over 0 dims"), (8, [1e-5], "over 8 dims"), (1, [-1e-5], "epsilon"), (1, [float("nan")], "epsilon"),
    (1, [], "epsilon"), (1, [1e-5, 1.], "epsilon")])
def test_attributes_that_make_no_sense_are_refused(g, rank, reals, match):
    from tenncor_amd import graph
    x = var(g, [4, 3])
    for op, args in (("LAYER_NORM", [x]), ("LAYER_NORM_DX", [x, x]), ("LAYER_NORM_DWEIGHT", [x, x])):
        with pytest.raises(graph.GraphError, match=match):
            g.functor(op, args, rank=rank, reals=reals)
    with pytest.raises(graph.GraphError, match="attribute"):
        g.functor("LAYER_NORM", [x], rank=1)


def test_operands_that_do_not_fit_are_refused(g, api):
    from tenncor_amd import graph
    x = var(g, [4, 3])
    for bad in ([3], [4, 3], [1]):
        with pytest.raises(graph.GraphError, match="weight or bias of shape"):
            api.layer_norm(x, var(g, bad))
        with pytest.raises(graph.GraphError, match="weight or bias of shape"):
            api.layer_norm(x, var(g, [4]), var(g, bad))
    with pytest.raises(graph.GraphError, match="4 arguments"):
        g.functor("LAYER_NORM", [x] + [var(g, [4])] * 3, rank=1, reals=[0.])
    with pytest.raises(graph.GraphError, match="incompatible shapes"):
        g.functor("LAYER_NORM_DX", [var(g, [4, 2]), x], rank=1, reals=[0.])
    with pytest.raises(graph.GraphError, match="1 arguments"):
        g.functor("LAYER_NORM_DX", [x], rank=1, reals=[0.])
    with pytest.raises(graph.GraphError, match="3 arguments"):
        g.functor("LAYER_NORM_DWEIGHT", [x, x, x], rank=1, reals=[0.])


def test_integers_are_not_normalised_and_mixed_types_are_cast(g, api):
    from tenncor_amd import capi, graph
    with pytest.raises(graph.GraphError, match="cannot LAYER_NORM integers"):
        api.layer_norm(var(g, [4, 3], np.int32))
    out = api.layer_norm(var(g, [4, 3], np.float32), var(g, [4], np.float64))
    assert out.dtype == capi.DOUBLE and g.opcode(g.args(out)[0]) == "CAST"


def test_gradients_are_one_node_each(g, api):
    x, w, b, up = var(g, [4, 3]), var(g, [4]), var(g, [4]), var(g, [4, 3])
    out = api.layer_norm(x, w, b, epsilon=0.5)
    dx, dw, db = (g.local_derivative(out, up, k) for k in range(3))
    assert [g.opcode(d) for d in (dx, dw, db)] == ["LAYER_NORM_DX", "LAYER_NORM_DWEIGHT", "REDUCE_SUM"]
    assert [a.id for a in g.args(dx)] == [up.id, x.id, w.id]
    assert [a.id for a in g.args(dw)] == [up.id, x.id]
    assert g.attr(dx, "reals") == g.attr(dw, "reals") == [0.5] and g.attr(dx, "rank") == g.attr(dw, "rank") == [1]
    assert g.attr(db, "rank_set") == list(range(1, 8))
    assert dw.shape == w.shape and db.shape == b.shape
    bare = api.layer_norm(x)
    assert [a.id for a in g.args(g.local_derivative(bare, up, 0))] == [up.id, x.id]


def test_the_gradient_nodes_have_no_derivative(g):
    from tenncor_amd import graph
    x = var(g, [4, 3])
    for op in ("LAYER_NORM_DX", "LAYER_NORM_DWEIGHT"):
        node = g.functor(op, [x, x], rank=1, reals=[0.])
        with pytest.raises(graph.GraphError, match="cannot derive " + op):
            g.local_derivative(node, var(g, node.shape), 0)


def test_every_bit_of_epsilon_tells_nodes_apart(g, api):
    """The clean-up merges equal nodes: two epsilons that print alike are not equal."""
    x = var(g, [4, 3])
    eps = np.float64(1e-5)
    near = np.nextafter(eps, 1)
    same, other = api.layer_norm(x, epsilon=eps), api.layer_norm(x, epsilon=near)
    again = api.layer_norm(x, epsilon=eps)
    roots, stats = g.optimize([same, other, again], rules=None, fold=False)
    assert roots[0].id != roots[1].id and stats["merged"] == 1


def test_it_is_a_launch_of_its_own_between_elementwise_groups(g, api):
    x, w, b = var(g, [64, 512]), var(g, [64]), var(g, [64])
    out = api.tanh(api.layer_norm(api.mul(x, 2.0), w, b))
    plan = g.launch_plan([out])
    assert sum(line.startswith("node LAYER_NORM") for line in plan) == 1
    # nothing that has no step of a batch is put into one
    small = api.tanh(api.layer_norm(api.mul(var(g, [4, 3]), 2.0)))
    assert all("LAYER_NORM" not in line for line in g.launch_plan([small]) if line.startswith("batch"))


class _Fake:
    """Stands in for a device tensor where only the checks run."""

    def __init__(self, shape, dtype=2):
        from tenncor_amd import capi
        self.shape, self.dtype, self.ctx, self.ptr = capi.shape8(shape), dtype, None, 0

    @property
    def n(self):
        from tenncor_amd import capi
        return capi.n_elems(self.shape)


def test_ops_check_their_arguments():
    from tenncor_amd import ops
    x = _Fake([4, 3])
    for weight, ndims in ((_Fake([3]), 1), (_Fake([4]), 2), (_Fake([4, 3]), 1)):
        with pytest.raises(ValueError, match="weight or bias"):
            ops.layer_norm(x, weight, ndims=ndims)
    with pytest.raises(ValueError, match="one type"):
        ops.layer_norm(x, _Fake([4], 1))
    for ndims in (0, 9):
        with pytest.raises(ValueError, match="over %d dims" % ndims):
            ops.layer_norm(x, ndims=ndims)
    with pytest.raises(ValueError, match="incompatible shapes"):
        ops.layer_norm_grad(_Fake([4, 2]), x)
    with pytest.raises(ValueError, match="of one type"):
        ops.layer_norm_grad(_Fake([4, 3], 1), x)
    kept = _Fake([1, 3])
    for mean, rstd in ((_Fake([1, 2]), kept), (kept, _Fake([4, 3])), (_Fake([1, 3], 1), kept), (kept, _Fake([1, 3], 1))):
        with pytest.raises(ValueError, match="for every row"):
            ops.layer_norm_grad(x, x, mean=mean, rstd=rstd)


def test_more_dims_than_there_are(g, api):
    for ndims in (0, 8, 257):
        with pytest.raises(ValueError, match="over %d dims" % ndims):
            api.layer_norm(var(g, [4, 3]), ndims=ndims)
