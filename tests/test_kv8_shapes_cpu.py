"""The numpy drivers of the 8-bit KV cache's operators refuse arrays that do not fit each other, before anything is sent to a GPU."""
import importlib

import numpy as np
import pytest

import kv8_oracle as plain


@pytest.fixture(scope="module")
def bind():
    return importlib.import_module("qwen3-tts-native_b200.ops")


def _ints(*shape):
    return np.zeros(shape, dtype=np.int32)


@pytest.mark.parametrize("args", [([1, 2], [1], _ints(2, 4), _ints(8)), ([1, 2], [1, 1], _ints(1, 4), _ints(8)), ([1, 2], [1, 1], _ints(8), _ints(8)),
                                  ([1, 2], [1, 1], _ints(2, 4), _ints(2, 4)), ([[1, 2]], [[1, 1]], _ints(2, 4), _ints(8))])
def test_page_tables(bind, args):
    with pytest.raises(ValueError, match="other arguments"):
        bind.page_tables(*args, 8)


@pytest.mark.parametrize("tokens,width,values,slots", [(3, 256, 3, 4), (4, 128, 4, 4), (4, 256, 3, 4), (4, 264, 4, 4)])
def test_append(bind, tokens, width, values, slots):
    planes = plain.cache(np.random.default_rng(1), 3, 2, 128, False)
    new = lambda n: np.zeros((n, width), dtype=np.uint16)  # noqa: E731
    with pytest.raises(ValueError, match="other arguments"):
        bind.kv8_append(*planes, new(tokens), new(values), np.arange(slots))


@pytest.mark.parametrize("width,rows,table,starts", [(200, 2, (2, 4), [0, 1, 2]), (256, 2, (1, 4), [0, 1, 2]), (256, 2, (8,), [0, 1, 2]),
                                                     (256, 2, (2, 4), [0, 2]), (256, 2, (2, 4), [0, 1, 2, 2])])
def test_attention(bind, width, rows, table, starts):
    planes = plain.cache(np.random.default_rng(1), 3, 2, 128, False)
    with pytest.raises(ValueError, match="other arguments"):
        bind.kv8_attention(np.zeros((2, width), dtype=np.uint16), *planes, _ints(*table), [5] * rows, starts)
