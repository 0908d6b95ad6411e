"""Calls of the 8-bit KV cache's operators beside those of test_gpu_kv8_attention.py."""
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
