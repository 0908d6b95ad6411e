"""Keys and values quantised into pages (q3t_launch_kv8_append) against a loop over pages and heads in fp32.  The definition fixes
every operation and its rounding, so codes and scales are equal to the bit."""
import ctypes as C

import numpy as np
import pytest

import kv8_oracle as plain

pytestmark = pytest.mark.gpu


def _check(ops, planes, k, v, slots, e4m3, count=None):
    got = ops.kv8_append(planes[0], planes[1], planes[2], planes[3], k, v, slots, e4m3=e4m3, count=count)
    used = slots if count is None else slots[:max(count, 0)]
    n = len(used)
    for i, new in ((0, k), (1, v)):
        codes, scales = plain.append_plane(planes[i], planes[i + 2], new[:n], used, e4m3)
        assert np.array_equal(got[i + 2], scales), "scales"
        same = got[i] == codes
        if e4m3:                                                              # zero has two codes
            same |= (got[i] & 0x7f == 0) & (codes & 0x7f == 0)
        assert same.all(), (i, np.argwhere(~same)[:4].tolist())
    return got


def _tokens(rng, count, width, size=1.0):
    rows = rng.standard_normal((count, width)) * np.exp(rng.uniform(-1, 1, (count, 1))) * size
    return plain.to_bf16(rows.astype(np.float32))


def _slots(rng, pages, held, new):
    """Slots of the new tokens of rows that hold `held`, over a page table of their own."""
    table = plain.tables_of(rng, [h + n for h, n in zip(held, new)], pages)
    return np.array([int(table[r, p // 16]) * 16 + p % 16 for r, (h, n) in enumerate(zip(held, new)) for p in range(h, h + n)], dtype=np.int64)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("heads,dim", [(8, 128), (1, 64), (3, 128), (2, 64)])
@pytest.mark.parametrize("held,new", [([0], [1]), ([5], [1]), ([15, 16, 17, 0], [1, 1, 1, 1]), ([0, 3, 30], [16, 29, 33]), ([7, 0], [100, 64])])
def test_rows_of_tokens(ops, e4m3, heads, dim, held, new):
    rng = np.random.default_rng(7 * heads + dim + sum(new))
    planes = plain.cache(rng, 24, heads, dim, e4m3)
    planes[2] *= np.float32(0.3)                                              # small enough that new tokens make scales grow
    slots = _slots(rng, 24, held, new)
    _check(ops, planes, _tokens(rng, len(slots), heads * dim), _tokens(rng, len(slots), heads * dim), slots, e4m3)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("heads", [2, 8, 16])
def test_windows_of_many_tokens(ops, heads, e4m3):
    """The kernel's three windows, which grow with tokens and heads: whole and broken pages, single tokens, padding between them."""
    rng = np.random.default_rng(11)
    dim, pages = 64, 400
    held = [int(x) for x in rng.integers(0, 40, 60)]
    new = [1 if rng.integers(0, 2) else int(rng.integers(1, 90)) for _ in held]
    new[-1] += max(0, 2111 - sum(new))
    slots = _slots(rng, pages, held, new)
    at = rng.choice(len(slots), 40, replace=False)
    for p in at:                                                              # whole pages of padding, so that no page stands apart
        page = slots[p] // 16
        if page >= 0:
            slots[slots // 16 == page] = -1 - int(rng.integers(0, 50))
    _check(ops, plain.cache(rng, pages, heads, dim, e4m3), _tokens(rng, len(slots), heads * dim), _tokens(rng, len(slots), heads * dim), slots, e4m3)


@pytest.mark.parametrize("e4m3", [False, True])
def test_token_by_token_and_again(ops, e4m3):
    """Scales only grow while a page fills, and the same token appended again changes nothing."""
    rng = np.random.default_rng(13)
    heads, dim = 2, 128
    planes = plain.cache(rng, 3, heads, dim, e4m3)
    k, v = (_tokens(rng, 20, heads * dim) for _ in range(2))
    for t in range(20):
        slots = np.array([16 + t if t < 16 else t - 16], dtype=np.int64)
        planes = _check(ops, planes, k[t:t + 1], v[t:t + 1], slots, e4m3)
        again = ops.kv8_append(*planes, k[t:t + 1], v[t:t + 1], slots, e4m3=e4m3)
        assert all(np.array_equal(a, b) for a, b in zip(planes, again))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("count", [0, 1, 6, 7, 50, -3])
def test_padding_and_a_count_on_the_device(ops, e4m3, count):
    rng = np.random.default_rng(17)
    planes = plain.cache(rng, 4, 2, 64, e4m3)
    slots = np.array([-1, 3, 4, -1, -7, 16, 63], dtype=np.int64)
    _check(ops, planes, _tokens(rng, 7, 128), _tokens(rng, 7, 128), slots, e4m3, count=min(count, 7) if count < 50 else 50)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("copies", [2, 40, 70])
def test_a_slot_named_again_keeps_the_last_token(ops, e4m3, copies):
    """Padded rows of a captured step often point at one slot."""
    rng = np.random.default_rng(copies)
    planes = plain.cache(rng, 4, 1, 128, e4m3)
    slots = np.array([37, 38] + [19] * copies + [18, 19, 20], dtype=np.int64)
    _check(ops, planes, _tokens(rng, len(slots), 128), _tokens(rng, len(slots), 128), slots, e4m3)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("size", [0.0, 1e-38, 1e-30, 1e30])
def test_sizes_from_nothing_to_the_largest(ops, e4m3, size):
    rng = np.random.default_rng(19)
    planes = plain.cache(rng, 3, 2, 64, e4m3)
    slots = np.arange(20, 40, dtype=np.int64)
    k = _tokens(rng, 20, 128, size)
    k[3, 5] = 0x7f7f                                                          # the largest bf16 beside them
    _check(ops, planes, k, _tokens(rng, 20, 128, size), slots, e4m3)


@pytest.mark.parametrize("e4m3", [False, True])
def test_what_is_not_finite(ops, q3t, e4m3):
    rng = np.random.default_rng(23)
    planes = plain.cache(rng, 3, 2, 64, e4m3)
    k, v = _tokens(rng, 20, 128), _tokens(rng, 20, 128)
    k[2, 7], k[2, 9], k[9, 100] = 0x7f80, 0xff80, 0xffc1                      # head 0 and head 1 of page 0
    before = q3t.library().q3t_kv8_nonfinite_count()
    _check(ops, planes, k, v, np.arange(4, 24, dtype=np.int64), e4m3)
    assert q3t.library().q3t_kv8_nonfinite_count() == before + 2


def test_slots_past_the_pool_are_left_out_and_counted(ops, q3t):
    rng = np.random.default_rng(29)
    planes = plain.cache(rng, 3, 2, 64, False)
    slots = np.array([48, 5, 2 ** 40, 2 ** 31 * 16 + 7, 17], dtype=np.int64)
    before = q3t.library().q3t_kv8_page_error_count()
    _check(ops, planes, _tokens(rng, 5, 128), _tokens(rng, 5, 128), slots, False)
    assert q3t.library().q3t_kv8_page_error_count() == before + 3


@pytest.mark.parametrize("e4m3", [False, True])
def test_packed_projections_pages_apart_and_offsets_past_32_bits(ops, q3t, e4m3):
    """Keys and values inside one packed projection, pages of a plane more than 2^31 bytes apart, on a stream of its own."""
    import torch
    rng = np.random.default_rng(31)
    heads, dim, pages, stride = 2, 64, 3, (1 << 31) + 4096
    kind = torch.float8_e4m3fn if e4m3 else torch.int8
    planes = plain.cache(rng, pages, heads, dim, e4m3)
    pool = torch.empty(2 * stride + 65536, dtype=torch.uint8, device="cuda")
    views = [torch.as_strided(pool[at:], (pages, heads, 16, dim), (stride, 16 * dim, dim, 1)) for at in (0, 16384)]
    scales = torch.zeros((pages, 2, heads), dtype=torch.float32, device="cuda")
    for i in range(2):
        views[i].copy_(torch.from_numpy(planes[i]).cuda())
        scales[:, i].copy_(torch.from_numpy(planes[i + 2]).cuda())
    c = ops.kv8_cache(views[0].view(kind), views[1].view(kind), scales[:, 0], scales[:, 1])
    slots = np.array([3, 4, 32, 33, 34, 21], dtype=np.int64)
    width = heads * dim
    packed = _tokens(rng, 6, 4 * width)
    dp, ds = torch.from_numpy(packed.view(np.int16)).cuda(), torch.from_numpy(slots).cuda()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    assert q3t.library().q3t_launch_kv8_append(C.byref(c), C.c_void_p(dp.data_ptr() + 4 * width), C.c_void_p(dp.data_ptr() + 6 * width),
                                               C.c_void_p(ds.data_ptr()), None, 6, 4 * width, 4 * width, C.c_void_p(stream.cuda_stream)) == 0
    stream.synchronize()
    for i in range(2):
        codes, want = plain.append_plane(planes[i], planes[i + 2], packed[:, (2 + i) * width:(3 + i) * width], slots, e4m3)
        got = views[i].cpu().numpy()
        assert ((got == codes) | ((got & 0x7f == 0) & (codes & 0x7f == 0))).all()
        assert np.array_equal(scales[:, i].cpu().numpy(), want)
