"""Attention over pages by blocks that leave their sums in memory: captured, side by side, over its queries."""
import numpy as np
import pytest

from pygpukit_b200.core.stream import CudaGraph, Stream, use_stream
from tests.test_gpu_paged import Step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,rows", [("bfloat16", 1), ("float16", 70), ("float32", 2)])
def test_blocks_that_are_no_cluster_captured_side_by_side_and_over_queries(dtype, rows):
    """two graphs of a call whose blocks leave their sums in memory, replayed at the same time; and outputs that take the queries' place"""
    s = Step([(9000, rows), (3, min(rows, 3))], 4, 1, 128, 64, dtype, "tree" if rows > 1 else "chain", seed=23)
    want = s.run()
    s.check(want)
    a = s.arrays()
    a["out"] = a["q"]
    s.call(a, weigh=False)
    assert np.array_equal(s.read(a)[0], want[0])
    sets, streams, graphs = [s.arrays() for _ in range(2)], [Stream() for _ in range(2)], []
    for x, st in zip(sets, streams):
        with use_stream(st):
            s.call(x, weigh=False)
            st.synchronize()
            g = CudaGraph()
            with g.capture(st):
                for _ in range(3):
                    s.call(x, weigh=False)
            graphs.append(g)
    for _ in range(4):
        for g, st in zip(graphs, streams):
            g.replay(st)
    for st in streams:
        st.synchronize()
    for x in sets:
        got = s.read(x)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
