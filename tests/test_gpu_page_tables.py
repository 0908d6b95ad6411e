"""Block tables and slot maps built on the GPU (q3t_launch_page_tables) against a loop over the rows.  Whole numbers: all equal."""
import ctypes as C

import numpy as np
import pytest

import kv8_oracle as plain

pytestmark = pytest.mark.gpu


def _case(rng, rows, longest, stride, spare, prompts, refuse=False):
    lengths = rng.integers(0, longest + 1, rows)
    changes = np.ones(rows, dtype=np.int64)
    for r in range(rows):
        kind = rng.integers(0, 6)
        if kind == 0:
            changes[r] = -lengths[r]
        elif kind == 1:
            changes[r] = -int(rng.integers(0, lengths[r] + 1))
        elif kind == 2 and prompts:
            changes[r] = int(rng.integers(1, prompts + 1))
        elif kind == 3:
            changes[r] = 0
        if refuse and rng.integers(0, 7) == 0:
            bad = rng.integers(0, 4)
            if bad == 0:
                lengths[r], changes[r] = -5, 7
            elif bad == 1:
                changes[r] = -lengths[r] - 1
            elif bad == 2:
                changes[r] = stride * 16 - lengths[r] + 1
            else:
                lengths[r], changes[r] = 2 ** 31 - 1, 2 ** 31 - 1
    held = [n if 0 <= n <= stride * 16 else 0 for n in lengths]
    used = sum(-(-int(n) // 16) for n in held)
    pages = used + spare
    table = plain.tables_of(rng, held, pages, stride)
    free = np.setdiff1d(np.arange(pages), table[table >= 0])
    stack = np.full(max(pages, 1), -99, dtype=np.int32)
    stack[:free.size] = rng.permutation(free)
    return lengths, changes, table, stack, free.size


def _check(got, want, table, stack, fill=-7):
    assert np.array_equal(got["status"], want["status"])
    assert np.array_equal(got["lengths"], want["lengths"])
    assert np.array_equal(got["starts"], want["starts"])
    assert np.array_equal(got["page_table"], want["page_table"])
    n = len(want["slots"])
    assert np.array_equal(got["positions"][:n], want["positions"]) and (got["positions"][n:] == fill).all()
    assert np.array_equal(got["slots"][:n], want["slots"]) and (got["slots"][n:] == fill).all()
    assert got["free_count"] == len(want["free"])
    assert np.array_equal(got["free_pages"][:len(want["free"])], want["free"])
    # (what lies above the new top and lay above the old one too is untouched)
    assert np.array_equal(got["free_pages"][len(want["free"]):], stack[len(want["free"]):])


@pytest.mark.parametrize("rows,longest,stride,spare,prompts,refuse", [
    (1, 0, 4, 4, 40, False), (1, 64, 4, 0, 0, False), (64, 2048, 160, 200, 0, False), (3, 15, 7, 1, 60, False),
    (37, 300, 64, 60, 500, True), (1000, 400, 96, 900, 700, True), (1025, 90, 12, 40, 60, True), (4096, 100, 40, 2000, 300, True),
    (512, 500, 40, 300, 0, True), (513, 500, 40, 300, 0, False)])
def test_against_a_loop_over_the_rows(ops, rows, longest, stride, spare, prompts, refuse):
    rng = np.random.default_rng(rows + longest)
    for _ in range(3):
        lengths, changes, table, stack, free = _case(rng, rows, longest, stride, spare, prompts, refuse)
        grown = int(np.clip(changes[changes < 2 ** 30], 0, None).sum())
        for capacity in (grown + 5, grown // 2, 0):
            want = plain.page_tables(lengths, changes, table, stack, free, capacity)
            _check(ops.page_tables(lengths, changes, table, stack, free, token_capacity=capacity), want, table, stack)


def test_pages_given_back_are_taken_in_the_same_launch(ops):
    table = np.array([[5, 2, 7], [1, 0, -1], [-1, -1, -1]], dtype=np.int32)
    stack = np.array([3, 9, 0, 0, 0, 0, 0, 0], dtype=np.int32)
    got = ops.page_tables([48, 17, 0], [-33, 16, 16], table, stack, 1)
    # row 0 keeps a page and gives back 2 and 7: the stack is 3, 2, 7; row 1 takes 7, row 2 takes 2
    assert got["page_table"].tolist() == [[5, 2, 7], [1, 0, 7], [2, -1, -1]] and got["free_count"] == 1
    _check(got, plain.page_tables([48, 17, 0], [-33, 16, 16], table, stack, 1, 32), table, stack)


def test_more_given_back_than_the_pool_holds_is_dropped(ops):
    table = np.array([[0, 1, 2, 3]], dtype=np.int32)
    stack = np.array([8, 9, -1], dtype=np.int32)
    got = ops.page_tables([64], [-64], table, stack, 2)
    assert got["free_count"] == 3 and got["free_pages"].tolist() == [8, 9, 0]


def test_free_count_outside_the_pool_is_clamped(ops):
    table = np.full((1, 4), -1, dtype=np.int32)
    stack = np.array([4, 5], dtype=np.int32)
    assert ops.page_tables([0], [64], table, stack, 99)["status"].tolist() == [plain.NO_PAGES]
    got = ops.page_tables([0], [32], table, stack, 99)
    assert got["page_table"][0].tolist() == [5, 4, -1, -1] and got["free_count"] == 0
    got = ops.page_tables([0], [1], table, stack, -3)
    assert got["status"].tolist() == [plain.NO_PAGES] and got["free_count"] == 0


@pytest.mark.parametrize("capacity", [5, 64, 5000])
def test_in_place_captured_and_replayed_on_another_stream(ops, q3t, capacity):
    """A step's tables captured once, lengths and stack advanced in place by every replay (one launch, or two)."""
    import torch
    lib = q3t.library()
    rows, stride, pages, steps = 5, 8, 40, 37
    rng = np.random.default_rng(3)
    lengths = np.array([0, 1, 15, 16, 40])
    table = plain.tables_of(rng, lengths, pages, stride)
    free = np.setdiff1d(np.arange(pages), table[table >= 0])
    stack = np.zeros(pages, dtype=np.int32)
    stack[:free.size] = free
    i32 = lambda a: torch.tensor(np.asarray(a, dtype=np.int32), device="cuda")  # noqa: E731
    held = dict(lengths=i32(lengths), changes=i32(np.ones(rows)), page_table=i32(table), free_pages=i32(stack), free_count=i32([free.size]),
                status=i32(np.zeros(rows)), token_starts=i32(np.zeros(rows + 1)), positions=i32(np.zeros(capacity)))
    slots = torch.zeros(capacity, dtype=torch.int64, device="cuda")
    d = ops.PageTablesDescC(rows=rows, page_table_stride=stride, pages=pages, token_capacity=capacity)
    d.struct_size = C.sizeof(d)
    for name, t in held.items():
        setattr(d, name, t.data_ptr())
    d.new_lengths, d.new_free_count, d.slots = held["lengths"].data_ptr(), held["free_count"].data_ptr(), slots.data_ptr()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        assert lib.q3t_launch_page_tables(C.byref(d), C.c_void_p(stream.cuda_stream)) == 0
    changes, count = np.ones(rows, dtype=int), free.size
    for step in range(steps):
        graph.replay()
        torch.cuda.synchronize()
        want = plain.page_tables(lengths, changes, table, stack, count, capacity)
        stack = held["free_pages"].cpu().numpy()
        _check(dict(status=held["status"].cpu().numpy(), lengths=held["lengths"].cpu().numpy(), starts=held["token_starts"].cpu().numpy(),
                    page_table=held["page_table"].cpu().numpy(), positions=held["positions"].cpu().numpy()[:len(want["slots"])],
                    slots=slots.cpu().numpy()[:len(want["slots"])], free_count=int(held["free_count"].item()), free_pages=stack), want, table, stack)
        lengths, table, count = want["lengths"], want["page_table"], len(want["free"])
