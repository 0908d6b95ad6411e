"""Refusals of the 8-bit KV cache's entry points (no GPU is touched) and the numpy forms the GPU tests compare with."""
import ctypes as C
import importlib

import numpy as np
import pytest

import kv8_oracle as plain

INVALID = 1                    # cudaErrorInvalidValue


@pytest.fixture(scope="module")
def bind():
    return importlib.import_module("qwen3-tts-native_b200.ops")


@pytest.fixture(scope="module")
def lib(q3t):
    return q3t.library()


def _cache(bind, **over):
    c = bind.Kv8CacheC(format=0, key_pages=4096, value_pages=8192, key_scales=256, value_scales=512, pages=4, key_value_heads=2, head_dimension=128)
    c.struct_size = C.sizeof(c)
    for k, v in over.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [dict(struct_size=8), dict(format=2), dict(format=-1), dict(key_pages=None), dict(value_pages=None), dict(key_scales=None),
              dict(value_scales=None), dict(key_pages=4104), dict(value_pages=8193), dict(key_scales=258), dict(pages=0), dict(key_value_heads=0),
              dict(key_value_heads=65), dict(head_dimension=32), dict(head_dimension=96), dict(head_dimension=256), dict(page_stride=4095),
              dict(page_stride=4104), dict(page_stride=-16), dict(scale_stride=1), dict(reserved=1)]


def _tables(bind, **over):
    d = bind.PageTablesDescC(rows=2, page_table_stride=4, pages=8, token_capacity=16)
    d.struct_size = C.sizeof(d)
    for name in ("lengths", "changes", "new_lengths", "page_table", "free_pages", "free_count", "new_free_count", "status", "token_starts"):
        setattr(d, name, 256)
    for k, v in over.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("over", [dict(struct_size=0), dict(rows=0), dict(rows=4097), dict(lengths=None), dict(changes=None), dict(new_lengths=None),
                                  dict(page_table=None), dict(free_pages=None), dict(free_count=None), dict(new_free_count=None), dict(status=None),
                                  dict(token_starts=None), dict(page_table_stride=0), dict(page_table_stride=2 ** 27), dict(pages=0),
                                  dict(token_capacity=-1), dict(reserved=3)])
def test_tables_refuse(bind, lib, over):
    assert lib.q3t_launch_page_tables(C.byref(_tables(bind, **over)), None) == INVALID
    assert lib.q3t_launch_page_tables(None, None) == INVALID


@pytest.mark.parametrize("over", BAD_CACHES)
def test_append_refuses_a_cache(bind, lib, over):
    p = C.c_void_p
    assert lib.q3t_launch_kv8_append(C.byref(_cache(bind, **over)), p(256), p(256), p(256), None, 1, 0, 0, None) == INVALID


@pytest.mark.parametrize("key,value,slots,tokens,ks,vs", [
    (None, 256, 256, 1, 0, 0), (256, None, 256, 1, 0, 0), (256, 256, None, 1, 0, 0), (256, 256, 256, 0, 0, 0), (256, 256, 256, -1, 0, 0),
    (264, 256, 256, 1, 0, 0), (256, 258, 256, 1, 0, 0), (256, 256, 260, 1, 0, 0), (256, 256, 256, 1, 248, 0), (256, 256, 256, 1, 260, 0),
    (256, 256, 256, 1, 0, 257), (256, 256, 256, 1, -256, 0)])
def test_append_refuses(bind, lib, key, value, slots, tokens, ks, vs):
    p = C.c_void_p
    assert lib.q3t_launch_kv8_append(C.byref(_cache(bind)), p(key), p(value), p(slots), None, tokens, ks, vs, None) == INVALID
    assert lib.q3t_launch_kv8_append(None, p(256), p(256), p(256), None, 1, 0, 0, None) == INVALID


def _attention(bind, held, **over):
    d = bind.Kv8AttentionDescC(rows=2, query_heads=4, page_table_stride=4, tokens=8, max_row_tokens=4, max_sequence_length=64, scratch=4096,
                               scratch_bytes=1 << 30)
    d.struct_size = C.sizeof(d)
    d.cache = C.addressof(held)
    for name in ("query", "output", "page_table", "lengths", "token_starts"):
        setattr(d, name, 4096)
    for k, v in over.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("over", [dict(struct_size=0), dict(rows=0), dict(rows=4097), dict(cache=None), dict(query=None), dict(output=None),
                                  dict(page_table=None), dict(lengths=None), dict(page_table_stride=0), dict(query_heads=0), dict(query_heads=3),
                                  dict(query_heads=130), dict(query_stride=504), dict(query_stride=516), dict(output_stride=513), dict(tokens=-1),
                                  dict(max_row_tokens=-1), dict(max_sequence_length=0), dict(max_sequence_length=65), dict(scale=-1.0),
                                  dict(scale=float("nan")), dict(query=4104), dict(output=4098), dict(output_f32=4100),
                                  dict(token_starts=None, tokens=1), dict(token_starts=None, max_row_tokens=0)])
def test_attention_refuses(bind, lib, over):
    d = _attention(bind, _cache(bind), **over)
    assert lib.q3t_kv8_attention_scratch_bytes(C.byref(d)) == 0
    assert lib.q3t_launch_kv8_attention(C.byref(d), None) == INVALID


@pytest.mark.parametrize("over", [dict(scratch=None), dict(scratch_bytes=0), dict(scratch=4100)])
def test_attention_refuses_a_scratch(bind, lib, over):
    c = _cache(bind)
    assert lib.q3t_kv8_attention_scratch_bytes(C.byref(_attention(bind, c))) > 0
    assert lib.q3t_launch_kv8_attention(C.byref(_attention(bind, c, **over)), None) == INVALID
    assert lib.q3t_launch_kv8_attention(None, None) == INVALID and lib.q3t_kv8_attention_scratch_bytes(None) == 0


def test_scratch_is_enough_for_smaller_launches(bind, lib):
    import random
    rng = random.Random(5)
    size = lambda high: int(round(2 ** rng.uniform(0, high)))  # noqa: E731
    for _ in range(400):
        heads, group, dim = rng.choice([1, 2, 8, 16]), rng.choice([1, 2, 8]), rng.choice([64, 128])
        c = _cache(bind, key_value_heads=heads, head_dimension=dim)
        rows, tokens, length = size(9), size(14), size(18)
        most = min(size(14), tokens)

        def need(rows, tokens, most, length):
            d = _attention(bind, c, rows=rows, query_heads=heads * group, page_table_stride=-(-length // 16), tokens=tokens, max_row_tokens=most,
                           max_sequence_length=length, query_stride=0, output_stride=0)
            return lib.q3t_kv8_attention_scratch_bytes(C.byref(d))
        whole = need(rows, tokens, most, length)
        for _ in range(6):
            less = [rng.randint(1, n) for n in (rows, tokens, most, length)]
            assert 0 < need(*less) <= whole


@pytest.mark.parametrize("over", BAD_CACHES)
def test_attention_refuses_a_cache(bind, lib, over):
    c = _cache(bind, **over)
    assert lib.q3t_launch_kv8_attention(C.byref(_attention(bind, c)), None) == INVALID


def test_nothing_to_do_launches_nothing(bind, lib):
    assert lib.q3t_launch_kv8_attention(C.byref(_attention(bind, _cache(bind), tokens=0)), None) == 0
    assert lib.q3t_launch_kv8_attention(C.byref(_attention(bind, _cache(bind), max_row_tokens=0)), None) == 0


def test_cache_descriptor_of_tensors(bind):
    import torch
    key = torch.zeros((3, 2, 16, 64), dtype=torch.int8)
    scales = torch.zeros((3, 2))
    c = bind.kv8_cache(key, key.clone(), scales, scales.clone())
    assert (c.format, c.pages, c.key_value_heads, c.head_dimension, c.page_stride, c.scale_stride) == (0, 3, 2, 64, 2048, 2)
    wide = torch.zeros((3, 2, 2, 16, 64), dtype=torch.float8_e4m3fn)
    assert bind.kv8_cache(wide[:, 0], wide[:, 1], scales, scales).page_stride == 4096
    for planes in ((key, wide[:, 0], scales, scales), (key, key.transpose(1, 2).contiguous().transpose(1, 2), scales, scales),
                   (key, key, scales.double(), scales), (key, key, scales, scales[:2]), (key.float(), key.float(), scales, scales),
                   (key[..., :8, :], key[..., :8, :], scales, scales)):
        with pytest.raises(ValueError):
            bind.kv8_cache(*planes)


def test_every_e4m3_code_is_its_own_nearest():
    codes = np.array([c for c in range(256) if c & 0x7f != 0x7f], dtype=np.uint8)
    assert np.array_equal(plain.encode(plain.E4M3[codes], True), codes)
    # halfway between two codes: the even one; beyond the last: the last
    low, high = plain.E4M3[0x40:0x48], plain.E4M3[0x41:0x49]
    assert np.array_equal(plain.encode((low + high) / 2, True) & 1, np.zeros(8, dtype=np.uint8))
    assert plain.encode(np.array([1e9, -500.0]), True).tolist() == [0x7e, 0xfe]
    assert plain.encode(np.array([0.5, 1.5, -2.5, 300.0]), False).view(np.int8).tolist() == [0, 2, -2, 127]


def test_append_keeps_what_is_held_and_grows_scales():
    rng = np.random.default_rng(5)
    codes, _, scales, _ = plain.cache(rng, 2, 1, 64, False)
    before = plain.decode(codes, False) * scales[:, :, None, None]
    new = plain.to_bf16(np.full((1, 64), 100.0, dtype=np.float32))
    after, grown = plain.append_plane(codes, scales, new, [16 + 9], False)
    assert grown[1, 0] == np.float32(100) / np.float32(127) and grown[0, 0] == scales[0, 0]
    values = plain.decode(after, False) * grown[:, :, None, None]
    assert np.abs(values[1, 0, :9] - before[1, 0, :9]).max() <= grown[1, 0] / 2 * 1.0001
    assert np.array_equal(after[1, 0, 10:], codes[1, 0, 10:]) and np.array_equal(after[0], codes[0])


def test_tables_by_hand():
    got = plain.page_tables([48, 17, 0], [-33, 16, 16], np.array([[5, 2, 7], [1, 0, -1], [-1, -1, -1]], dtype=np.int32), [3, 0, 0, 0], 1, 99)
    assert got["page_table"].tolist() == [[5, 2, 7], [1, 0, 7], [2, -1, -1]] and got["free"] == [3]
    assert got["starts"].tolist() == [0, 0, 16, 32] and got["slots"][:2].tolist() == [1, 2] and got["slots"][15] == 7 * 16
