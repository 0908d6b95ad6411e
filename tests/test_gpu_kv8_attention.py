"""Attention over an 8-bit paged cache (q3t_launch_kv8_attention) against the formula in 64 bits (tests/kv8_oracle.py, which derives the
tolerance).  The bf16 output may be half a bf16 step further off: 2^-9 of the next power of two, 2^-8 of the value at most.

Which kernel takes a row depends on the bounds that the host gives, so most tests run with page tables of several widths: as wide as
the rows need (a CTA or a cluster a segment, prompts in one part), FEW_TOKENS pages (ranges of pages for every warp) and LONG pages
(prompts of many tokens in parts)."""
import ctypes as C

import numpy as np
import pytest

import kv8_oracle as plain

pytestmark = pytest.mark.gpu
FEW_TOKENS, LONG = 520, 70000
ROOMS = pytest.mark.parametrize("room", [None, FEW_TOKENS, LONG])


def _query(rng, count, heads, dim, size=1.0):
    return plain.to_bf16((rng.standard_normal((count, heads * dim)) * size).astype(np.float32))


def _compare(out, f32, want, tol, empty=None):
    shape = want.shape
    if f32 is not None:
        off = np.abs(f32.reshape(shape) - want)
        assert (off <= tol).all(), (off / np.maximum(tol, 1e-300)).max()
    off = np.abs(plain.from_bf16(out).astype(np.float64).reshape(shape) - want)
    assert (off <= tol + (np.abs(want) + tol) * 2.0 ** -8).all(), (off / np.maximum(tol + np.abs(want) * 2.0 ** -8, 1e-300)).max()


def _run(ops, rng, heads, dim, group, lengths, new, e4m3, **more):
    pages = sum(-(-max(n, 0) // 16) for n in lengths) + 3
    spread = more.pop("spread", 0.5)
    size = more.pop("size", 1.0)
    planes = plain.cache(rng, pages, heads, dim, e4m3, spread)
    table = plain.tables_of(rng, lengths, pages, more.pop("room", None))
    starts = None if new is None else np.concatenate([[0], np.cumsum(new)])
    count = len(lengths) if new is None else int(starts[-1])
    q = _query(rng, count, heads * group, dim, size)
    out, f32 = ops.kv8_attention(q, *planes, table, lengths, starts, e4m3=e4m3, want_f32=True, **more)
    want, tol = plain.attention(q, planes, table, lengths, starts, e4m3, more.get("max_seq"), more.get("scale"))
    _compare(out, f32, want, tol)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dim", [128, 64])
@pytest.mark.parametrize("heads,group", [(8, 2), (1, 1), (2, 4), (1, 8), (2, 7), (1, 16), (1, 33)])
@pytest.mark.parametrize("room", [None, FEW_TOKENS])
def test_single_tokens(ops, e4m3, dim, heads, group, room):
    rng = np.random.default_rng(heads * 100 + group)
    _run(ops, rng, heads, dim, group, [1, 15, 16, 17, 300, 128, 129, 1025, 0], None, e4m3, room=room)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("length", [1, 127, 2048, 2049, 5000, 40000])
@pytest.mark.parametrize("room", [None, 2600])
def test_one_row_of_any_length(ops, e4m3, length, room):
    _run(ops, np.random.default_rng(length), 2, 128, 2, [length], None, e4m3, room=room)


@pytest.mark.parametrize("rows", [2, 64, 300, 1500])
@pytest.mark.parametrize("room", [None, FEW_TOKENS])
def test_many_rows(ops, rows, room):
    rng = np.random.default_rng(rows)
    _run(ops, rng, 1, 64, 2, [int(n) for n in rng.integers(0, 200, rows)], None, rows % 4 == 0, room=room)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("heads,dim,group,rows,longest,new", [
    (1, 128, 2, 4, 5000, None), (2, 64, 1, 16, 7000, None), (8, 128, 1, 8, 4096, None), (8, 128, 2, 16, 2000, None), (4, 64, 8, 60, 900, None),
    (8, 128, 2, 50, 500, None), (2, 128, 4, 4, 3000, [3, 1, 9, 0]), (8, 64, 2, 3, 1500, [30, 4, 11])])
def test_clusters_of_every_size(ops, e4m3, heads, dim, group, rows, longest, new):
    """8, 8, 4, 2 and 1 CTAs a segment, these in two rounds as well, with blocks that some rows do not have; among the rows one of nothing and one of one page."""
    rng = np.random.default_rng(rows + longest)
    lengths = [int(n) for n in rng.integers(20, longest + 1, rows)]
    lengths[0] = longest
    if new is None:
        lengths[1:3] = [0, 9]
    _run(ops, rng, heads, dim, group, lengths, new, e4m3)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("heads,dim,group,lengths,new", [(8, 128, 2, [2100], [64]), (8, 64, 1, [1200, 90, 1500], [40, 60, 9]), (1, 128, 16, [9000, 40], [20, 7])])
def test_rows_of_many_columns_over_a_long_context(ops, e4m3, heads, dim, group, lengths, new):
    """Too few tokens to fill the SMs with prompts' blocks: the ranges of the short rows' kernel, several blocks of columns a row."""
    _run(ops, np.random.default_rng(sum(lengths)), heads, dim, group, lengths, new, e4m3)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("heads,dim,group,lengths,new", [
    (1, 128, 16, [3000], [200]), (2, 64, 2, [8200], [260]), (1, 64, 4, [8200, 130, 40, 20], [230, 120, 40, 60]), (1, 128, 8, [5000, 0, 4097], [33, 0, 190])])
def test_prompts_in_parts(ops, e4m3, heads, dim, group, lengths, new):
    """Two to eight parts of a long context; rows of fewer steps than parts and one that is shorter than its new tokens."""
    _run(ops, np.random.default_rng(sum(lengths) + 1), heads, dim, group, lengths, new, e4m3)


@pytest.mark.parametrize("heads,group,lengths,new", [(64, 1, [300], [300]), (64, 1, [310, 300], [300, 300])])
def test_more_prompt_blocks_than_sms(ops, heads, group, lengths, new):
    """Blocks of 128 columns and of 256."""
    _run(ops, np.random.default_rng(len(new)), heads, 64, group, lengths, new, len(new) == 1)


@pytest.mark.parametrize("heads,lengths,new,room", [(2, [700, 500], None, None), (2, [700, 500], None, FEW_TOKENS), (2, [900], [200], LONG), (8, [900], [200], None)])
@pytest.mark.parametrize("e4m3", [False, True])
def test_scores_that_grow_along_the_context(ops, heads, lengths, new, room, e4m3):
    """Keys a fifth larger from page to page: references are outgrown again and again, late ones by far."""
    rng = np.random.default_rng(79)
    planes = plain.cache(rng, 120, heads, 128, e4m3)
    table = plain.tables_of(rng, lengths, 120, room)
    for r, n in enumerate(lengths):
        ids = table[r, :-(-n // 16)]
        planes[2][ids] *= (1.2 ** np.arange(len(ids)) * 0.02).astype(np.float32)[:, None]
    starts = None if new is None else np.concatenate([[0], np.cumsum(new)])
    q = _query(rng, len(lengths) if new is None else sum(new), heads * 2, 128)
    out, f32 = ops.kv8_attention(q, *planes, table, lengths, starts, e4m3=e4m3, want_f32=True)
    want, tol = plain.attention(q, planes, table, lengths, starts, e4m3)
    _compare(out, f32, want, tol)


@pytest.mark.parametrize("heads,lengths,new,room", [(2, [700, 500], None, None), (2, [700, 500], None, FEW_TOKENS), (2, [900, 64], [90, 30], LONG), (8, [400], [140], None)])
@pytest.mark.parametrize("zeros,size", [(z, n) for z in ("first", "most", "all") for n in (1.0, 1e8, 1e-18, 1e-27)] + [("none", 1e36), ("none", 1e-30)])
def test_pages_of_zeros_weigh_what_their_scores_say(ops, heads, lengths, new, room, zeros, size):
    """Values of nothing have the scale 2^-126, and their tokens a share of the sum all the same; values from the smallest to the largest."""
    e4m3 = zeros in ("first", "none")
    rng = np.random.default_rng(97)
    planes = plain.cache(rng, 120, heads, 128, e4m3)
    table = plain.tables_of(rng, lengths, 120, room)
    planes[3] *= np.float32(size)
    for r, n in enumerate(lengths):
        ids = table[r, :-(-n // 16)]
        none = {"none": ids[:0], "first": ids[:len(ids) // 2], "most": ids[np.arange(len(ids)) % 9 != 4], "all": ids}[zeros]
        planes[1][none], planes[3][none] = 0, plain.SMALLEST
    starts = None if new is None else np.concatenate([[0], np.cumsum(new)])
    q = _query(rng, len(lengths) if new is None else sum(new), heads * 2, 128, 2.0)
    out, f32 = ops.kv8_attention(q, *planes, table, lengths, starts, e4m3=e4m3, want_f32=True)
    want, tol = plain.attention(q, planes, table, lengths, starts, e4m3)
    _compare(out, f32, want, tol)


@pytest.mark.parametrize("heads,lengths,new,room", [(2, [300, 200], None, None), (2, [300, 200], None, FEW_TOKENS), (2, [300], [150], LONG), (8, [300], [150], None)])
@pytest.mark.parametrize("value", [0x7f80, 0xffc0])
def test_queries_that_are_not_finite_stay_in_their_rows(ops, heads, lengths, new, room, value):
    rng = np.random.default_rng(83)
    planes = plain.cache(rng, 40, heads, 128, False)
    table = plain.tables_of(rng, lengths, 40, room)
    starts = None if new is None else np.concatenate([[0], np.cumsum(new)])
    count = len(lengths) if new is None else sum(new)
    q = _query(rng, count, heads * 2, 128)
    want, tol = plain.attention(q, planes, table, lengths, starts, False)
    bad = np.zeros(want.shape[:2], dtype=bool)
    for token, head in ((0, 1), (count - 1, heads * 2 - 1)):
        q[token, head * 128 + 5] = value
        bad[token, head] = True
    out, f32 = ops.kv8_attention(q, *planes, table, lengths, starts, want_f32=True)
    f32 = f32.reshape(want.shape)
    assert np.isnan(f32[bad]).all()
    assert (np.abs(f32 - want)[~bad] <= tol[~bad]).all()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("heads,dim,group", [(2, 128, 2), (1, 64, 4), (2, 64, 1), (1, 128, 5)])
@ROOMS
@pytest.mark.parametrize("lengths,new", [([5, 100, 33], [5, 5, 5]), ([700, 20, 0, 9], [1, 17, 0, 9]), ([64, 300], [64, 3]), ([2, 40], [4, 40])])
def test_ragged_new_tokens(ops, e4m3, heads, dim, group, lengths, new, room):
    """Drafts, prompts, rows without new tokens, and one that is shorter than its new tokens (its first ones get zeros)."""
    _run(ops, np.random.default_rng(sum(lengths) + group), heads, dim, group, lengths, new, e4m3, room=room)


@pytest.mark.parametrize("e4m3", [False, True])
@ROOMS
@pytest.mark.parametrize("heads,dim,group,lengths,new", [
    (8, 128, 2, [140, 33, 32, 350], [140, 16, 17, 129]), (8, 64, 1, [65, 500, 257], [65, 300, 257]), (2, 128, 2, [200], [200]), (1, 128, 2, [129, 400], [129, 130]), (1, 64, 4, [257], [257]), (1, 128, 8, [700], [90]), (1, 64, 1, [600, 1, 350], [300, 1, 129]),
    (1, 128, 3, [301], [170]), (1, 128, 16, [130], [67])])
def test_prompts_and_chunks(ops, e4m3, heads, dim, group, lengths, new, room):
    _run(ops, np.random.default_rng(sum(lengths) + group), heads, dim, group, lengths, new, e4m3, room=room)


@pytest.mark.parametrize("e4m3", [False, True])
@ROOMS
@pytest.mark.parametrize("new", [None, [40, 140]])
@pytest.mark.parametrize("spread,size", [(6.0, 1.0), (0.1, 30.0), (0.5, 1e-30)])
def test_scales_and_queries_of_any_size(ops, e4m3, new, spread, size, room):
    """Page scales a factor of e^12 apart, scores that leave one token standing, queries that leave none."""
    _run(ops, np.random.default_rng(41), 2, 128, 2, [500, 333], new, e4m3, spread=spread, size=size, room=room)


@pytest.mark.parametrize("new", [None, [1, 150]])
def test_scale_of_the_scores_and_a_cut_context(ops, q3t, new):
    rng = np.random.default_rng(43)
    before = q3t.library().q3t_attention_range_error_count()
    _run(ops, rng, 2, 128, 2, [300, 260], new, False, scale=0.02)
    assert q3t.library().q3t_attention_range_error_count() == before
    _run(ops, rng, 2, 128, 2, [300, 260], new, False, max_seq=272)
    assert q3t.library().q3t_attention_range_error_count() == before + 1


@pytest.mark.parametrize("heads,group,length,new,most", [(16, 2, 300, 140, 272), (1, 16, 9000, 64, 8992), (2, 2, 300, 20, 272)])
def test_a_cut_context_of_one_row(ops, q3t, heads, group, length, new, most):
    """A prompt alone is one launch (or, in parts, two), which counts for itself; a row of no new tokens has nothing to write."""
    before = q3t.library().q3t_attention_range_error_count()
    _run(ops, np.random.default_rng(most), heads, 64, group, [length], [new], False, max_seq=most)
    assert q3t.library().q3t_attention_range_error_count() == before + 1
    rng = np.random.default_rng(most + 1)
    planes = plain.cache(rng, 570, heads, 64, False)
    q = _query(rng, new, heads * group, 64)
    out, _ = ops.kv8_attention(q, *planes, plain.tables_of(rng, [length], 570), [length], [0, 0], max_row_tokens=new, fill=0x1234)
    assert (out == 0x1234).all()


@pytest.mark.parametrize("e4m3", [False, True])
@ROOMS
@pytest.mark.parametrize("new", [None, [1, 1, 150]])
def test_what_lies_behind_the_last_token_does_not_matter(ops, e4m3, new, room):
    """Slots past the end hold NaN codes (e4m3) or -128, pages past the end lie anywhere."""
    rng = np.random.default_rng(47)
    lengths = [21, 250, 199]
    planes = plain.cache(rng, 40, 2, 128, e4m3)
    table = plain.tables_of(rng, lengths, 40, room or 20)
    starts = None if new is None else np.concatenate([[0], np.cumsum(new)])
    q = _query(rng, 3 if new is None else sum(new), 4, 128)
    clean = ops.kv8_attention(q, *planes, table, lengths, starts, e4m3=e4m3)[0]
    for r, n in enumerate(lengths):
        for plane in planes[:2]:
            plane[table[r, n // 16], :, n % 16:] = 0x7f if e4m3 else 0x80
    dirty = ops.kv8_attention(q, *planes, table, lengths, starts, e4m3=e4m3)[0]
    assert np.array_equal(clean, dirty)


@ROOMS
@pytest.mark.parametrize("new", [None, [1, 140, 2]])
def test_bad_pages_are_left_out_and_counted(ops, q3t, new, room):
    rng = np.random.default_rng(53)
    lengths = [100, 250, 31]
    planes = plain.cache(rng, 40, 2, 128, False)
    table = plain.tables_of(rng, lengths, 40, room)
    table[0, 2], table[1, 0], table[1, 9], table[2, 0], table[2, 1] = 40, -1, 2 ** 31 - 1, -2 ** 31, 41
    starts = None if new is None else np.concatenate([[0], np.cumsum(new)])
    q = _query(rng, 3 if new is None else sum(new), 4, 128)
    before = q3t.library().q3t_kv8_page_error_count()
    out, f32 = ops.kv8_attention(q, *planes, table, lengths, starts, want_f32=True)
    assert q3t.library().q3t_kv8_page_error_count() >= before + 5
    want, tol = plain.attention(q, planes, table, lengths, starts, False)
    _compare(out, f32, want, tol)
    assert not plain.from_bf16(out[-1]).any()                                 # nothing left of row 2


def test_rows_behind_the_last_token_keep_their_bits(ops):
    rng = np.random.default_rng(59)
    planes = plain.cache(rng, 10, 2, 64, False)
    table = plain.tables_of(rng, [50, 60], 10)
    q = _query(rng, 40, 4, 64)
    out, _ = ops.kv8_attention(q, *planes, table, [50, 60], [0, 3, 33], max_row_tokens=30, fill=0x1234)
    assert (out[33:] == 0x1234).all() and not (out[:33] == 0x1234).all(axis=1).any()


def test_bounds_of_the_host_cut_what_the_device_finds(ops, q3t):
    """Starts beyond `tokens`, descending starts and rows of more tokens than max_row_tokens stay inside the buffers and are counted."""
    rng = np.random.default_rng(61)
    planes = plain.cache(rng, 10, 2, 64, False)
    table = plain.tables_of(rng, [50, 60], 10)
    q = _query(rng, 20, 4, 64)
    for starts, most, written in (([0, 5, 400], 20, range(20)), ([0, 12, 20], 8, [*range(8), *range(12, 20)]), ([0, 9, 3], 20, range(9)), ([-4, 5, 9], 20, range(9))):
        before = q3t.library().q3t_attention_range_error_count()
        out, _ = ops.kv8_attention(q, *planes, table, [50, 60], starts, max_row_tokens=most, fill=0x1234)
        touched = ~(out == 0x1234).all(axis=1)
        assert touched.nonzero()[0].tolist() == list(written)
        assert q3t.library().q3t_attention_range_error_count() > before


@pytest.mark.parametrize("e4m3", [False, True])
def test_strides_a_shared_pool_and_offsets_past_32_bits(ops, q3t, e4m3):
    import torch
    rng = np.random.default_rng(67)
    heads, dim, group, pages, stride = 2, 128, 2, 3, (1 << 31) + 8192
    kind = torch.float8_e4m3fn if e4m3 else torch.int8
    planes = plain.cache(rng, pages, heads, dim, e4m3)
    pool = torch.empty(2 * stride + 65536, dtype=torch.uint8, device="cuda")
    views = [torch.as_strided(pool[at:], (pages, heads, 16, dim), (stride, 16 * dim, dim, 1)) for at in (0, 16384)]
    scales = torch.zeros((pages, 5, heads), dtype=torch.float32, device="cuda")
    for i in range(2):
        views[i].copy_(torch.from_numpy(planes[i]).cuda())
        scales[:, i].copy_(torch.from_numpy(planes[i + 2]).cuda())
    c = ops.kv8_cache(views[0].view(kind), views[1].view(kind), scales[:, 0], scales[:, 1])
    width = heads * group * dim
    for new in ([1], [37]):
        length, count = [47], sum(new)
        table = np.array([[2, 0, 1]], dtype=np.int32)
        q = _query(rng, count, heads * group, dim)
        wide = np.zeros((count, width + 24), dtype=np.uint16)
        wide[:, 8:8 + width] = q
        dq = torch.from_numpy(wide.view(np.int16)).cuda()
        do = torch.full((count, width + 40), 7, dtype=torch.int16, device="cuda")
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        held = [i32(table), i32(length), i32([0, count])]
        d = ops.Kv8AttentionDescC(rows=1, query_heads=heads * group, page_table_stride=3, tokens=count, max_row_tokens=count, max_sequence_length=48,
                                  query_stride=width + 24, output_stride=width + 40)
        d.struct_size = C.sizeof(d)
        d.cache, d.query, d.output = C.addressof(c), dq.data_ptr() + 16, do.data_ptr() + 32
        d.page_table, d.lengths, d.token_starts = (t.data_ptr() for t in held)
        size = q3t.library().q3t_kv8_attention_scratch_bytes(C.byref(d))
        scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
        d.scratch, d.scratch_bytes = scratch.data_ptr(), size
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        assert q3t.library().q3t_launch_kv8_attention(C.byref(d), C.c_void_p(stream.cuda_stream)) == 0
        stream.synchronize()
        got = do.cpu().numpy().view(np.uint16)
        want, tol = plain.attention(q, planes, table, length, [0, count], e4m3)
        _compare(got[:, 16:16 + width], None, want, tol)
        assert (got[:, :16] == 7).all() and (got[:, 16 + width:] == 7).all()


def test_the_same_call_gives_the_same_bits(ops):
    rng = np.random.default_rng(71)
    lengths = [3000, 700, 1, 5000]
    planes = plain.cache(rng, 560, 2, 128, False)
    table = plain.tables_of(rng, lengths, 560)
    for new in (None, [1, 100, 1, 300], [1, 100, 1, 500]):                  # (ranges; the same; prompts in parts)
        starts = None if new is None else np.concatenate([[0], np.cumsum(new)])
        q = _query(rng, 4 if new is None else sum(new), 4, 128)
        first = ops.kv8_attention(q, *planes, table, lengths, starts, want_f32=True)
        for _ in range(4):
            again = ops.kv8_attention(q, *planes, table, lengths, starts, want_f32=True)
            assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])


class _Call:
    """A launch of its own: descriptor, buffers and, unless one is lent, scratch."""
    def __init__(self, ops, lib, planes, table, lengths, starts, q, group, scratch=None):
        import torch
        i32 = lambda a: torch.tensor(np.asarray(a, dtype=np.int32), device="cuda")  # noqa: E731
        heads, dim = planes[0].shape[1], planes[0].shape[3]
        self.lib, self.planes = lib, ops._planes(*planes, False)
        self.cache = ops.kv8_cache(*self.planes)
        self.held = [i32(table), i32(lengths), i32(starts), torch.from_numpy(q.view(np.int16)).cuda()]
        self.out = torch.zeros(q.shape, dtype=torch.int16, device="cuda")
        self.desc = d = ops.Kv8AttentionDescC(rows=len(lengths), query_heads=heads * group, page_table_stride=table.shape[1], tokens=len(q),
                                              max_row_tokens=int(np.diff(starts).max()), max_sequence_length=16 * table.shape[1])
        d.struct_size = C.sizeof(d)
        d.cache, d.output = C.addressof(self.cache), self.out.data_ptr()
        d.page_table, d.lengths, d.token_starts, d.query = (t.data_ptr() for t in self.held)
        size = lib.q3t_kv8_attention_scratch_bytes(C.byref(d))
        self.scratch = torch.empty(size, dtype=torch.uint8, device="cuda") if scratch is None else scratch
        assert self.scratch.numel() >= size
        d.scratch, d.scratch_bytes = self.scratch.data_ptr(), self.scratch.numel()

    def launch(self, stream):
        assert self.lib.q3t_launch_kv8_attention(C.byref(self.desc), C.c_void_p(stream.cuda_stream)) == 0

    def result(self):
        return self.out.cpu().numpy().copy()


def _calls(ops, lib, scratch=None):
    """Single tokens, a few tokens over long rows, and prompts in parts beside single tokens."""
    rng = np.random.default_rng(89)
    calls = []
    for lengths, new in (([900, 3000, 40], [1, 1, 1]), ([9000, 700], [12, 30]), ([5000, 4100, 60], [700, 1, 60])):
        planes = plain.cache(rng, 700, 2, 128, False)
        q = _query(rng, sum(new), 4, 128)
        calls.append(_Call(ops, lib, planes, plain.tables_of(rng, lengths, 700, 600), lengths, np.concatenate([[0], np.cumsum(new)]), q, 2, scratch))
    return calls


def test_two_streams_at_once(ops, q3t):
    import torch
    first, second = _calls(ops, q3t.library()), _calls(ops, q3t.library())[::-1]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for call in first:
        call.launch(streams[0])
    torch.cuda.synchronize()
    want = [call.result() for call in first]
    for call in first:
        call.out.zero_()
    torch.cuda.synchronize()
    for _ in range(10):
        for a, b in zip(first, second):
            a.launch(streams[0])
            b.launch(streams[1])
    torch.cuda.synchronize()
    for call, other, right in zip(first, second[::-1], want):
        assert np.array_equal(call.result(), right) and np.array_equal(other.result(), right)


def test_captured_graphs_that_share_a_scratch(ops, q3t):
    """One scratch for launches of every kind, in two graphs that are replayed in turn."""
    import torch
    lib = q3t.library()
    alone = _calls(ops, lib)
    scratch = max((call.scratch for call in alone), key=lambda t: t.numel())
    scratch.fill_(0xa5)
    calls = _calls(ops, lib, scratch)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for call in alone:
        call.launch(stream)
        torch.cuda.synchronize()
    graphs = []
    for order in ((0, 1, 2), (2, 0, 1)):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            for i in order:
                calls[i].launch(stream)
    for n in range(6):
        for call in calls:
            call.out.zero_()
        torch.cuda.synchronize()
        for _ in range(3):
            graphs[n % 2].replay()
        torch.cuda.synchronize()
        for call, right in zip(calls, alone):
            assert np.array_equal(call.result(), right.result())


@pytest.mark.parametrize("e4m3", [False, True])
def test_a_decoder_s_steps_together(ops, q3t, e4m3):
    """Tables, append and attention as a decoder runs them: prompts, then steps replayed from one graph on another stream, requests that end
    and come in between.  The cache against the append's definition, the attention against the formula over that cache."""
    import torch
    lib = q3t.library()
    rng = np.random.default_rng(73)
    rows, heads, dim, group, stride, pages, capacity = 4, 2, 128, 2, 16, 40, 320
    i32 = lambda a: torch.tensor(np.asarray(a, dtype=np.int32), device="cuda")  # noqa: E731
    planes = plain.cache(rng, pages, heads, dim, e4m3)
    dplanes = ops._planes(*planes, e4m3)
    cache = ops.kv8_cache(*dplanes)
    held = dict(lengths=i32(np.zeros(rows)), changes=i32(np.zeros(rows)), page_table=i32(np.full((rows, stride), -1)),
                free_pages=i32(rng.permutation(pages)), free_count=i32([pages]), status=i32(np.zeros(rows)), token_starts=i32(np.zeros(rows + 1)),
                positions=i32(np.zeros(capacity)))
    slots = torch.zeros(capacity, dtype=torch.int64, device="cuda")
    t = ops.PageTablesDescC(rows=rows, page_table_stride=stride, pages=pages, token_capacity=capacity)
    t.struct_size = C.sizeof(t)
    for name, tensor in held.items():
        setattr(t, name, tensor.data_ptr())
    t.new_lengths, t.new_free_count, t.slots = held["lengths"].data_ptr(), held["free_count"].data_ptr(), slots.data_ptr()
    width = heads * dim
    packed = torch.zeros((capacity, (group + 2) * width), dtype=torch.int16, device="cuda")
    out = torch.zeros((capacity, group * width), dtype=torch.int16, device="cuda")

    def attention(tokens, most):
        d = ops.Kv8AttentionDescC(rows=rows, query_heads=heads * group, page_table_stride=stride, tokens=tokens, max_row_tokens=most,
                                  max_sequence_length=stride * 16, query_stride=packed.shape[1])
        d.struct_size = C.sizeof(d)
        d.cache, d.query, d.output = C.addressof(cache), packed.data_ptr(), out.data_ptr()
        d.page_table, d.lengths, d.token_starts = (held[n].data_ptr() for n in ("page_table", "lengths", "token_starts"))
        size = lib.q3t_kv8_attention_scratch_bytes(C.byref(d))
        scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
        d.scratch, d.scratch_bytes = scratch.data_ptr(), size
        return d, scratch

    def step(desc, tokens, stream):
        s = C.c_void_p(stream.cuda_stream)
        assert lib.q3t_launch_page_tables(C.byref(t), s) == 0
        count = held["token_starts"].data_ptr() + 4 * rows
        assert lib.q3t_launch_kv8_append(C.byref(cache), C.c_void_p(packed.data_ptr() + 2 * group * width),
                                         C.c_void_p(packed.data_ptr() + 2 * (group + 1) * width), C.c_void_p(slots.data_ptr()), C.c_void_p(count),
                                         tokens, packed.shape[1], packed.shape[1], s) == 0
        assert lib.q3t_launch_kv8_attention(C.byref(desc[0]), s) == 0

    stream = torch.cuda.Stream()
    big, small = attention(capacity, capacity), attention(rows, 1)
    step(big, capacity, stream)                                               # (no tokens: everything set up ahead of the capture)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        step(small, rows, stream)
    lengths, table = np.zeros(rows, dtype=int), np.full((rows, stride), -1, dtype=np.int32)
    stack, count = held["free_pages"].cpu().numpy(), pages
    plans = [[150, 3, 0, 17]] + [[1, 1, 0, 1]] * 15 + [[1, -18, 40, 1]] + [[1, 0, 1, 1]] * 9 + [[-170, 60, 1, -5]] + [[0, 1, 1, 1]] * 7
    for changes in plans:
        single = max(changes) <= 1
        want = plain.page_tables(lengths, changes, table, stack, count, rows if single else capacity)
        n = len(want["slots"])
        rows_new = plain.to_bf16(rng.standard_normal((capacity, packed.shape[1])).astype(np.float32))
        packed.copy_(torch.from_numpy(rows_new.view(np.int16)))
        held["changes"].copy_(i32(changes))
        torch.cuda.synchronize()
        if single:
            graph.replay()
        else:
            step(big, capacity, stream)
        torch.cuda.synchronize()
        lengths, table = want["lengths"], want["page_table"]
        stack, count = held["free_pages"].cpu().numpy(), len(want["free"])
        assert np.array_equal(held["lengths"].cpu().numpy(), lengths) and np.array_equal(held["page_table"].cpu().numpy(), table)
        assert np.array_equal(slots.cpu().numpy()[:n], want["slots"])
        for i in range(2):
            planes[i], planes[i + 2] = plain.append_plane(planes[i], planes[i + 2], rows_new[:n, (group + i) * width:(group + i + 1) * width], want["slots"], e4m3)
            assert np.array_equal(plain.decode(dplanes[i].view(torch.uint8).cpu().numpy(), e4m3), plain.decode(planes[i], e4m3))
            assert np.array_equal(dplanes[i + 2].cpu().numpy(), planes[i + 2])
        expect, tol = plain.attention(rows_new[:n, :group * width], planes, table, lengths, want["starts"], e4m3)
        _compare(out[:n].cpu().numpy().view(np.uint16), None, expect, tol)
