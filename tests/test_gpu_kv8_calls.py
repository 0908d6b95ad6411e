"""Calls of the 8-bit KV cache's operators beside those of test_gpu_kv8_attention.py."""
import importlib.util
import os
import subprocess
import sys

import numpy as np
import pytest

import kv8_oracle as plain
from test_gpu_kv8_attention import LONG, _compare, _query, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [128, 64])
@pytest.mark.parametrize("heads,group,new,room", [(64, 1, [33, 63], None), (16, 3, [37, 50], None), (16, 1, [129, 161, 255], None), (16, 7, [75], None),
                                                  (2, 1, [33, 63], LONG), (2, 3, [37, 50], LONG), (2, 1, [131, 255], LONG), (1, 7, [75], LONG)])
def test_warps_whose_last_columns_are_not_there(ops, dim, heads, group, new, room):
    """Prompts, in one part and in several, whose columns end anywhere in a warp of 32: what it loads together it stores in part."""
    lengths = [n + 100 * i for i, n in enumerate(new)]
    _run(ops, np.random.default_rng(sum(new) + dim), heads, dim, group, lengths, new, dim == 64, room=room)


@pytest.mark.parametrize("heads,group,dim,new,length", [(8, 2, 128, 256, 256), (8, 2, 64, 256, 500), (8, 1, 128, 512, 512), (1, 64, 64, 64, 64)])
def test_a_prompt_of_512_blocks_of_columns_is_a_prompt_however_short(ops, heads, group, dim, new, length):
    """With a bound of 1,024 tokens kv8_prompt.cu has it; the sums of the kernel of few new tokens run in another order, so equal bits say that
    a tight bound does not send it there, where it takes a fifth longer."""
    rng = np.random.default_rng(length + new)
    planes = plain.cache(rng, 40, heads, dim, False)
    table = plain.tables_of(rng, [length], 40, 64)
    q = _query(rng, new, heads * group, dim)
    tight, loose = (ops.kv8_attention(q, *planes, table, [length], [0, new], max_seq=bound, want_f32=True) for bound in (length, 1024))
    want, tol = plain.attention(q, planes, table, [length], [0, new], False)
    _compare(*tight, want, tol)
    assert np.array_equal(tight[0], loose[0]) and np.array_equal(tight[1], loose[1])


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


# a block that is lost, in a process of its own: others look for an error count of zero
LOST = """
import sys
sys.path[:0] = [{tests!r}, {root!r}]
import importlib
import numpy as np
import kv8_oracle as plain
q3t = importlib.import_module("qwen3-tts-native_b200")
ops = importlib.import_module("qwen3-tts-native_b200.ops")
lib = q3t.library()
rng = np.random.default_rng(3)
heads, group, dim = {heads}, 2, 64
lengths, new = {lengths}, {new}
starts = np.concatenate([[0], np.cumsum(new)])
planes = plain.cache(rng, 900, heads, dim, False)
table = plain.tables_of(rng, lengths, 900, {room})
q = plain.to_bf16(rng.standard_normal((sum(new), heads * group * dim)).astype(np.float32))
call = lambda: ops.kv8_attention(q, *planes, table, lengths, starts, fill=0x1234)[0].reshape(len(q), heads, group * dim)
want = call()
assert lib.q3t_kernel_error_count() == 0
lib.q3t_test_kv8_lose_block({block})
got = call()
assert lib.q3t_kernel_error_count() == 1
lib.q3t_test_kv8_lose_block(-1)
lost = np.zeros(got.shape[:2], dtype=bool)
lost[{tokens}, {head}] = True
assert (got[lost] == 0x1234).all(), "rows of the lost block were written"
assert np.array_equal(got[~lost], want[~lost])
assert np.array_equal(call(), want) and lib.q3t_kernel_error_count() == 1
"""


@pytest.mark.parametrize("heads,lengths,new,room,block,tokens,head", [
    # one part an item: blocks of 128 columns (64 tokens), the last tokens' and first head's first
    (16, [300, 40], [300, 40], None, 1, slice(256, 300), 1), (16, [300, 40], [300, 40], None, 16 * 5, slice(300, 340), 0),
    # eight parts an item, of which one of the first head's second block (tokens 128 .. 199) or one of the second row's is lost
    (2, [5000, 4100], [200, 60], LONG, 5, slice(128, 200), 0), (2, [5000, 4100], [200, 60], LONG, 8 * 4 + 8, slice(200, 260), 1)])
def test_what_a_block_that_gave_up_does_not_write(heads, lengths, new, room, block, tokens, head):
    here = os.path.dirname(os.path.abspath(__file__))
    code = LOST.format(tests=here, root=os.path.dirname(here), heads=heads, lengths=lengths, new=new, room=room, block=block,
                       tokens="slice(%d, %d)" % (tokens.start, tokens.stop), head=head)
    ran = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert ran.returncode == 0, ran.stderr[-2000:]


@pytest.mark.parametrize("heads,group,lengths,new,room", [
    (2, 2, [100, 250, 31], None, None), (2, 2, [3000, 250, 31], None, None), (2, 2, [100, 250, 31], None, 520), (8, 2, [2000, 900, 700] + [300] * 60, None, None),
    (2, 2, [300, 260, 31], [40, 90, 1], None), (16, 2, [300, 260, 31], [140, 90, 1], None), (16, 2, [500], [300], None),
    (2, 2, [5000, 4100, 60], [200, 60, 1], LONG), (2, 2, [9000], [300], None), (4, 2, [3000, 2100], [30, 9], None)])
def test_a_bad_page_is_counted_once(ops, q3t, heads, group, lengths, new, room):
    """However many heads, blocks of columns, warps and parts come by it."""
    rng = np.random.default_rng(sum(lengths))
    pages = sum(-(-n // 16) for n in lengths) + 3
    planes = plain.cache(rng, pages, heads, 64, False)
    table = plain.tables_of(rng, lengths, pages, room)
    bad = 0
    for r, n in enumerate(lengths[:3]):
        for page in {0, 2, -(-n // 16) // 2, -(-n // 16) - 1}:
            if page < -(-n // 16):
                table[r, page] = rng.choice([-1, pages, 2 ** 31 - 1, -2 ** 31])
                bad += 1
    starts = None if new is None else np.concatenate([[0], np.cumsum(new)])
    q = _query(rng, len(lengths) if new is None else sum(new), heads * group, 64)
    before, waits = q3t.library().q3t_kv8_page_error_count(), q3t.library().q3t_kernel_error_count()
    out, f32 = ops.kv8_attention(q, *planes, table, lengths, starts, want_f32=True)
    assert q3t.library().q3t_kv8_page_error_count() == before + bad and q3t.library().q3t_kernel_error_count() == waits
    want, tol = plain.attention(q, planes, table, lengths, starts, False)
    _compare(out, f32, want, tol)


@pytest.mark.parametrize("e4m3", [False, True])
def test_a_refused_draft_leaves_its_scale_until_the_page_begins_anew(ops, e4m3):
    rng = np.random.default_rng(17)
    planes = plain.cache(rng, 2, 1, 64, e4m3)
    tokens = lambda count, size: plain.to_bf16((rng.standard_normal((count, 64)) * size).astype(np.float32))  # noqa: E731
    first, large, small = tokens(6, 1.0), tokens(3, 50.0), tokens(3, 1.0)
    slots = lambda a, b: np.arange(16 + a, 16 + b, dtype=np.int64)  # noqa: E731
    held = ops.kv8_append(*planes, first, first, slots(0, 6), e4m3=e4m3)
    drafted = ops.kv8_append(*held, large, large, slots(6, 9), e4m3=e4m3)
    taken = ops.kv8_append(*drafted, small, small, slots(6, 9), e4m3=e4m3)            # the draft's slots, filled anew
    for i in range(2):
        assert drafted[i + 2][1, 0] > 5 * held[i + 2][1, 0] and taken[i + 2][1, 0] == drafted[i + 2][1, 0]
        assert np.array_equal(taken[i][1, :, :6], drafted[i][1, :, :6])
    again = ops.kv8_append(*taken, first, first, slots(0, 6), e4m3=e4m3)              # from the first slot on
    for i in range(2):
        assert again[i + 2][1, 0] == held[i + 2][1, 0] and np.array_equal(again[i][1, :, :6], held[i][1, :, :6])
