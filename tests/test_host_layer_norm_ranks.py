"""Numbers of dims of a LAYER_NORM node that a rank of 8 bits would take for others."""
import numpy as np
import pytest


@pytest.mark.parametrize("rank", [257, -255, 256, -1, 1 << 40, (1 << 40) + 1])
@pytest.mark.parametrize("op,count", [("LAYER_NORM", 1), ("LAYER_NORM_DX", 2), ("LAYER_NORM_DWEIGHT", 2)])
def test_numbers_beyond_a_rank_are_refused(rank, op, count):
    from tenncor_amd import graph
    g = graph.Graph()
    x = g.variable(np.arange(12, dtype=np.float32), [4, 3], "x")
    with pytest.raises(graph.GraphError, match="over %d dims" % rank):
        g.functor(op, [x] * count, rank=rank, reals=[1e-5])
    g.close()
