"""Calls of the 8-bit KV cache's operators beside those of test_gpu_kv8_attention.py."""
import importlib.util
import os

import numpy as np
import pytest

from test_gpu_kv8_attention import LONG, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [128, 64])
@pytest.mark.parametrize("heads,group,new,room", [(64, 1, [33, 63], None), (16, 3, [37, 50], None), (16, 1, [129, 161, 255], None), (16, 7, [75], None),
                                                  (2, 1, [33, 63], LONG), (2, 3, [37, 50], LONG), (2, 1, [131, 255], LONG), (1, 7, [75], LONG)])
def test_warps_whose_last_columns_are_not_there(ops, dim, heads, group, new, room):
    """Prompts, in one part and in several, whose columns end anywhere in a warp of 32: what it loads together it stores in part."""
    lengths = [n + 100 * i for i, n in enumerate(new)]
    _run(ops, np.random.default_rng(sum(new) + dim), heads, dim, group, lengths, new, dim == 64, room=room)


def test_a_measured_case_goes_to_the_stream_that_is_current():
    """What a state of perf/operators.py keeps of its call serves every stream: one that ran is captured, and the capture runs nothing."""
    import torch
    spec = importlib.util.spec_from_file_location("operators", os.path.join(os.path.dirname(__file__), "..", "perf", "operators.py"))
    cases = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(cases)
    cases.own = True
    state = cases.prepare({"kind": "attend", "format": "int8", "rows": 3, "shortest": 20, "longest": 90, "new": 1, "query_heads": 4, "heads": 2, "dim": 64}, 5)
    want = cases.run(state).clone()
    torch.cuda.synchronize()
    state["output"].zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        cases.run(state)
    torch.cuda.synchronize()
    assert want.any() and not state["output"].any()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(state["output"], want)
