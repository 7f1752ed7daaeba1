"""What the token mixers' entries refuse before they touch a device."""
import ctypes

import pytest


def cache(q8, pages=4, page_size=16, kv_heads=2, head_dim=64, fmt="bf16", **kw):
    c = q8.KVCache(4096, 8192, pages, page_size, kv_heads, head_dim,
                   *((256, 512) if fmt == "q8" else (None, None))).memref()
    for name, value in kw.items():
        setattr(c, name, value)
    return c


def batch(q8, sequences=3, max_pages=2, **kw):
    b = q8.KVBatch(256, 512, 768, sequences, max_pages).memref()
    for name, value in kw.items():
        setattr(b, name, value)
    return b


def status(q8, c, b):
    fn = q8.lib().llmcp_q8_test_kv_check
    fn.argtypes, fn.restype = [ctypes.c_void_p] * 2, ctypes.c_int
    return fn(ctypes.byref(c) if c is not None else None, ctypes.byref(b) if b is not None else None)


@pytest.mark.parametrize("kw", [
    {}, {"fmt": "q8"}, {"head_dim": 128}, {"head_dim": 256}, {"page_size": 1}, {"page_size": 7},
    {"page_size": 1 << 20, "pages": 1023}, {"kv_heads": 1024}, {"pages": (1 << 31) // 32 - 1}])
def test_caches_taken(q8, kw):
    assert status(q8, cache(q8, **kw), batch(q8)) == q8.OK


@pytest.mark.parametrize("kw", [
    {"head_dim": 32}, {"head_dim": 96}, {"head_dim": 512}, {"page_size": 0}, {"page_size": -16},
    {"page_size": (1 << 20) + 1}, {"kv_heads": 0}, {"kv_heads": 1025}, {"pages": 0}, {"pages": -1},
    {"pages": 1 << 26}, {"pages": 1 << 62}, {"keys": 4104}, {"values": 8194}])
def test_caches_declined(q8, kw):
    assert status(q8, cache(q8, **kw), batch(q8)) == q8.DECLINED


@pytest.mark.parametrize("kw", [
    {"keys": None}, {"values": None}, {"format": 2}, {"format": -1}, {"key_scales": 256},
    {"value_scales": 256}, {"fmt": "q8", "key_scales": None}, {"fmt": "q8", "value_scales": None}])
def test_caches_invalid(q8, kw):
    assert status(q8, cache(q8, **kw), batch(q8)) == q8.EINVAL


def test_batches(q8):
    assert status(q8, cache(q8), batch(q8, sequences=65536)) == q8.OK
    assert status(q8, cache(q8), batch(q8, max_pages=(1 << 26) - 1)) == q8.OK
    for kw in ({"sequences": 0}, {"sequences": -1}, {"sequences": 65537}, {"max_pages": 0},
               {"max_pages": 1 << 26}, {"max_pages": -4}):
        assert status(q8, cache(q8), batch(q8, **kw)) == q8.DECLINED
    for name in ("row_starts", "lengths", "page_table"):
        assert status(q8, cache(q8), batch(q8, **{name: None})) == q8.EINVAL
    assert status(q8, None, batch(q8)) == q8.EINVAL
    assert status(q8, cache(q8), None) == q8.EINVAL


def heads(q8, bf16, ptr=4096, sizes=(5, 2, 64), strides=(128, 64, 1), offset=0):
    fn = q8.lib().llmcp_q8_test_heads
    fn.argtypes, fn.restype = [ctypes.c_void_p, ctypes.c_int32], ctypes.c_int
    d = q8.heads_memref(ptr, 1, 1, 1)
    d.offset = offset
    for i in range(3):
        d.sizes[i], d.strides[i] = sizes[i], strides[i]
    return fn(ctypes.byref(d), int(bf16))


@pytest.mark.parametrize("bf16", [False, True])
def test_rows_of_heads(q8, bf16):
    ok, no = q8.OK, q8.DECLINED
    per = 8 if bf16 else 4
    assert heads(q8, bf16) == ok
    assert heads(q8, bf16, strides=(512, 64 + per, 1)) == ok
    assert heads(q8, bf16, offset=per) == ok
    assert heads(q8, bf16, sizes=(0, 2, 64)) == ok
    assert heads(q8, bf16, sizes=(1, 2, 64), strides=(3, 64, 1)) == ok  # one row: no stride
    assert heads(q8, bf16, sizes=(5, 1, 64), strides=(64, 3, 1)) == ok  # one head: none
    assert heads(q8, bf16, ptr=None) == no
    assert heads(q8, bf16, ptr=4096 + 2) == no
    assert heads(q8, bf16, offset=1) == no
    assert heads(q8, bf16, strides=(128, 64, 2)) == no
    assert heads(q8, bf16, strides=(128, 63, 1)) == no
    assert heads(q8, bf16, strides=(128, 65, 1)) == no
    assert heads(q8, bf16, strides=(129, 64, 1)) == no
    assert heads(q8, bf16, strides=(64, 64, 1)) == no
    assert heads(q8, bf16, strides=(-128, 64, 1)) == no
    assert heads(q8, bf16, sizes=(-1, 2, 64)) == no
    assert heads(q8, bf16, sizes=(5, 0, 64)) == no
    assert heads(q8, bf16, sizes=((1 << 23) + 1, 2, 64)) == no
    assert heads(q8, bf16, sizes=(5, 1025, 64), strides=(1025 * 64, 64, 1)) == no


def test_null_contexts(q8):
    L, x = q8.lib(), q8.heads_memref(4096, 1, 2, 64)
    c, b = cache(q8), batch(q8)
    p = ctypes.byref
    for t in ("", "_bf16"):
        assert getattr(L, "llmcp_q8_kv_write" + t)(None, p(x), p(x), p(b), p(c)) == q8.EINVAL
        assert getattr(L, "llmcp_q8_kv_read" + t)(None, p(c), p(b), p(x), p(x)) == q8.EINVAL
        assert getattr(L, "llmcp_q8_attention" + t)(None, p(x), p(c), p(b), 1.0, p(x)) == q8.EINVAL
        assert getattr(L, "llmcp_q8_delta_rule" + t)(None, p(x), p(x), p(x), None, None, 1.0, 1, 0.0,
                                                     None, 1, None, None, p(x)) == q8.EINVAL
