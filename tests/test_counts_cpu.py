"""Error counters that add up what several kernels counted: one of them that cannot be read is never lost in the sum."""
import importlib

import pytest
import torch

COUNTERS = ["q3t_kernel_error_count", "q3t_attention_range_error_count", "q3t_kv8_page_error_count", "q3t_kv8_nonfinite_count"]


@pytest.mark.skipif(torch.cuda.is_available(), reason="every counter can be read where there is a GPU")
@pytest.mark.parametrize("name", COUNTERS)
def test_a_count_that_cannot_be_read_says_so(name):
    lib = importlib.import_module("qwen3-tts-native_b200").library()
    assert getattr(lib, name)() & 0xffffffff == 0xffffffff
