"""CPU checks of the largest calls that the paged cache's C ABI takes, as its header states them: at the limit a workspace size
(nothing is launched), one above it the refusal."""

import ctypes
import os
import re

import pytest

import _attnres_hip as H
from test_cache_host import HEADER, _cache

pytestmark = pytest.mark.skipif(not os.path.exists(H.LIB_PATH), reason="libattnres_hip.so not built")
INT32_MAX = 2 ** 31 - 1


def limit(name):
    text = re.search(rf"#define ATTNRES_CACHE_MAX_{name} +(.*?) +/\*", open(HEADER).read())[1]
    return int(eval(text.replace("/", "//"), {"INT32_MAX": INT32_MAX}))


def attend(cache, tokens, q_heads):
    """(workspace bytes, code, message)"""
    lib = H.load()
    d = H.CacheAttendDesc(tokens=tokens, q_heads=q_heads, scale=0.125, q=0x6000, q_batch_stride=1, q_head_stride=1, q_token_stride=1,
                          decay=1.0)
    n = lib.attnres_cache_attend_workspace_size(ctypes.byref(cache), ctypes.byref(d))
    # (without a workspace the call ends at the host)
    code = lib.attnres_cache_attend(ctypes.byref(cache), ctypes.byref(d), 0x9000, None, 0, None)
    return n, code, lib.attnres_last_error().decode()


def test_values():
    """What the code was built with and the kernels' 32-bit counts hold."""
    assert [limit(n) for n in ("HEADS", "APPENDED", "QUERIES", "PIECES", "EVICTED", "KEPT")] == [
        2 ** 20, INT32_MAX, 2 ** 23, INT32_MAX // 2, 2 ** 21, INT32_MAX]


@pytest.mark.parametrize("batch,tokens,q_heads", [(64, 4096, 32), (1, 2 ** 20, 8), (2 ** 20, 1, 8), (1, 1, 2 ** 20)])
def test_queries(batch, tokens, q_heads):
    most = limit("QUERIES")
    assert batch * tokens * q_heads <= most
    cache = _cache(batch=batch, table_pages=1 << 10)  # (a table short enough for all of them: the pieces have their own limit)
    n, code, _ = attend(cache, tokens, q_heads)
    assert n > 0 and code == -4
    if batch * tokens * q_heads == most:
        n, code, text = attend(cache, tokens + 1, q_heads)
        assert n == 0 and code == -2 and "too many queries" in text


def test_pieces():
    # 2 key / value heads, 4 query heads, 1 token: one block of rows a head; 1 << 23 units of 128 tokens in the longest table
    cache = _cache(batch=63, page_size=1 << 10, table_pages=1 << 20)
    assert 63 * 2 * (1 << 23) <= limit("PIECES")
    assert attend(cache, 1, 4)[0] > 0
    cache.batch = 64
    n, code, text = attend(cache, 1, 4)
    assert 64 * 2 * (1 << 23) > limit("PIECES") and n == 0 and code == -2 and "too many tokens" in text


@pytest.mark.parametrize("name", ["batch", "kv_heads", "q_heads"])
def test_heads(name):
    most = limit("HEADS")
    kw = dict(batch=1, kv_heads=1, q_heads=1)
    for n, fine in ((most, True), (most + 1, False)):
        kw.update({name: n, **({"q_heads": n} if name == "kv_heads" else {})})
        size, code, text = attend(_cache(batch=kw["batch"], kv_heads=kw["kv_heads"], table_pages=1 << 12), 1, kw["q_heads"])
        assert (size > 0) == fine and (fine or (code == -1 and name in text and str(most) in text))


def test_appended_heads():
    lib = H.load()
    d = H.CacheAppendDesc(tokens=(limit("APPENDED") // 8) + 1, q_heads=4, table_dtype=0, qkv=0x6000, batch_stride=512, token_stride=512,
                          sin=0x7000, cos=0x8000, table_rows=8, table_row_stride=32)
    c = _cache(batch=1)
    assert lib.attnres_cache_append(ctypes.byref(c), ctypes.byref(d), 0x9000, None, None) == -2
    assert "too many" in lib.attnres_last_error().decode()


def test_evicted_heads():
    lib = H.load()

    def size(batch, table_pages, budget):
        c = _cache(weights=0x5000, batch=batch, kv_heads=2, page_size=16, table_pages=table_pages, table_stride=table_pages)
        n = lib.attnres_cache_evict_workspace_size(ctypes.byref(c), budget, 0)
        code = lib.attnres_cache_evict(ctypes.byref(c), 0x6000, 1 << 20, budget, 0, 0x7000, 0x8000, None, 0, None)
        return n, code, lib.attnres_last_error().decode()

    # four slices of 8192 tokens a head
    assert (1 << 18) * 2 * 4 == limit("EVICTED")
    assert size(1 << 18, 2048, 100)[:2] == ((1 << 21) * 3080 * 4, -4)
    n, code, text = size((1 << 18) + 1, 2048, 100)
    assert n == 0 and code == -2 and "too many" in text
    # places kept
    assert size(128, 2048, (limit("KEPT") + 1) // 256 - 1)[1] == -4
    n, code, text = size(128, 2048, (limit("KEPT") + 1) // 256)
    assert n == 0 and code == -2 and "too many" in text
