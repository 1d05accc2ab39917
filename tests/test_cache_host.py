"""CPU checks of the paged cache's operators: the C ABI's exports, struct layouts and refusals (nothing is launched), and the
Python functions' refusals of tensors that are not on a GPU."""

import ctypes
import os
import re
import subprocess

import pytest
import torch

import _attnres_hip as H
import attnres_ops as ops
from cache_util import Cache, attend_ref, evict_ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "attnres_cache.h")
needs_lib = pytest.mark.skipif(not os.path.exists(H.LIB_PATH), reason="libattnres_hip.so not built")
STRUCTS = ((H.CacheDesc, "attnres_cache_desc"), (H.CacheAppendDesc, "attnres_cache_append_desc"),
           (H.CacheAttendDesc, "attnres_cache_attend_desc"))


@needs_lib
def test_library_exports_every_declared_symbol():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(attnres_[a-z0-9_]+)\s*\(", text)))
    assert names == sorted(["attnres_cache_append", "attnres_cache_attend_workspace_size", "attnres_cache_attend",
                            "attnres_cache_evict", "attnres_cache_evict_workspace_size"])
    nm = subprocess.run(["nm", "-D", "--defined-only", H.LIB_PATH], capture_output=True, text=True).stdout
    for n in names:
        assert re.search(rf"\bT {n}\b", nm), n


def test_ctypes_structs_match_the_header(tmp_path):
    lines = [f'  printf("{n} sizeof %zu\\n", sizeof({n}));' for _, n in STRUCTS]
    lines += [f'  printf("{n} {f} %zu\\n", offsetof({n}, {f}));' for cls, n in STRUCTS for f, _ in cls._fields_]
    c, exe = tmp_path / "p.c", tmp_path / "p"
    c.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"attnres_cache.h\"\nint main(void) {\n" +
                 "\n".join(lines) + "\n  return 0;\n}\n")
    subprocess.run(["gcc", "-I", os.path.dirname(HEADER), str(c), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    lay = {tuple(line.split()[:2]): int(line.split()[2]) for line in out.strip().splitlines()}
    for cls, name in STRUCTS:
        assert ctypes.sizeof(cls) == lay[(name, "sizeof")]
        for f, _ in cls._fields_:
            assert getattr(cls, f).offset == lay[(name, f)], (name, f)


def _desc(cls, base, kw):
    d = cls(**base)
    for k, v in kw.items():
        if hasattr(d, k):
            setattr(d, k, v)
    return d


def _cache(**kw):
    return _desc(H.CacheDesc, dict(dtype=1, kv_heads=2, head_dim=64, page_size=16, pages=8, k=0x10000, v=0x20000, page_stride=2048,
                                   head_stride=1024, slot_stride=64, batch=2, block_table=0x3000, table_stride=4, table_pages=4,
                                   cached=0x4000), kw)


CACHE_REFUSALS = [
    (dict(dtype=7), -1, "dtype"), (dict(kv_heads=0), -1, "kv_heads"), (dict(head_dim=0), -1, "head_dim"),
    (dict(head_dim=258), -2, "head_dim"), (dict(page_size=0), -1, "page_size"), (dict(batch=-1), -1, "batch"),
    (dict(pages=-1), -1, "pages"), (dict(pages=1 << 31), -1, "pages"), (dict(table_pages=-1), -1, "table_pages"),
    (dict(table_pages=(1 << 26) + 1), -2, "table_pages"), (dict(cached=0), -1, "NULL"), (dict(block_table=0), -1, "NULL"),
    (dict(table_stride=-1), -1, "table_stride"), (dict(k=0), -1, "NULL"), (dict(v=0), -1, "NULL"),
    (dict(page_stride=-1), -1, "stride"), (dict(slot_stride=-2), -1, "stride"),
    (dict(weights=0x5000, weight_head_stride=-1), -1, "weight")]


@needs_lib
@pytest.mark.parametrize("kw,code,word", CACHE_REFUSALS + [
    (dict(table_dtype=2), -1, "table dtype"), (dict(tokens=-1), -1, "tokens"), (dict(q_heads=0), -1, "q_heads"),
    (dict(head_dim=63), -1, "even"), (dict(qkv=0), -1, "NULL"), (dict(sin=0), -1, "NULL"), (dict(cos=0), -1, "NULL"),
    (dict(batch_stride=-1), -1, "stride"), (dict(table_rows=0), -1, "table_rows"), (dict(table_row_stride=31), -1, "table_row_stride")])
def test_append_refusals(kw, code, word):
    lib = H.load()
    d = _desc(H.CacheAppendDesc, dict(tokens=1, q_heads=4, qk_norm=1, norm_eps=1e-7, table_dtype=0, qkv=0x6000, batch_stride=512,
                                      token_stride=512, sin=0x7000, cos=0x8000, table_rows=8, table_row_stride=32), kw)
    c = _cache(**kw)
    assert lib.attnres_cache_append(ctypes.byref(c), ctypes.byref(d), 0x9000, None, None) == code
    assert word in lib.attnres_last_error().decode()
    assert lib.attnres_cache_append(None, ctypes.byref(d), 0x9000, None, None) == -1


@needs_lib
@pytest.mark.parametrize("kw,code,word", CACHE_REFUSALS + [
    (dict(tokens=-1), -1, "tokens"), (dict(q_heads=3), -1, "q_heads"), (dict(q_heads=0), -1, "q_heads"),
    (dict(scale=float("inf")), -1, "scale"), (dict(scale=float("nan")), -1, "scale"), (dict(scale=-2e38), -1, "scale"), (dict(q=0), -1, "NULL"),
    (dict(q_token_stride=-1), -1, "stride"), (dict(weights=0x5000, tokens=2), -1, "single"),
    (dict(weights=0x5000, decay=1.5), -1, "decay"), (dict(weights=0x5000, decay=float("nan")), -1, "decay"),
    (dict(tokens=1 << 30), -2, "too many")])
def test_attend_refusals(kw, code, word):
    lib = H.load()
    d = _desc(H.CacheAttendDesc, dict(tokens=1, q_heads=4, scale=0.125, q=0x6000, q_batch_stride=256, q_head_stride=64,
                                      q_token_stride=64, decay=1.0), kw)
    c = _cache(**kw)
    assert lib.attnres_cache_attend(ctypes.byref(c), ctypes.byref(d), 0x9000, 0x100000, 1 << 30, None) == code
    assert word in lib.attnres_last_error().decode()
    assert lib.attnres_cache_attend_workspace_size(ctypes.byref(c), ctypes.byref(d)) == 0


@needs_lib
def test_attend_workspace():
    lib = H.load()
    d = H.CacheAttendDesc(tokens=1, q_heads=4, scale=0.125, q=0x6000, q_batch_stride=256, q_head_stride=64, q_token_stride=64, decay=1.0)
    c = _cache(weights=0x5000)
    n = lib.attnres_cache_attend_workspace_size(ctypes.byref(c), ctypes.byref(d))
    assert n > 0
    for ws, size in ((None, n), (0x100000, n - 1), (0x100010, n)):
        assert lib.attnres_cache_attend(ctypes.byref(c), ctypes.byref(d), 0x9000, ws, size, None) == -4
        assert "workspace" in lib.attnres_last_error().decode()
    assert lib.attnres_cache_attend(ctypes.byref(c), ctypes.byref(d), None, 0x100000, n, None) == -1
    d.tokens = 0
    assert lib.attnres_cache_attend(ctypes.byref(c), ctypes.byref(d), None, None, 0, None) == 0


@needs_lib
@pytest.mark.parametrize("kw,code,word", CACHE_REFUSALS + [
    (dict(budget=0), -1, "budget"), (dict(budget=1 << 31), -1, "budget"), (dict(recent=-1), -1, "recent"), (dict(recent=33), -1, "recent"),
    (dict(new=None), -1, "NULL"), (dict(kept=None), -1, "NULL"), (dict(left=None), -1, "NULL"), (dict(weights=0), -1, "weights"),
    (dict(new_stride=1), -1, "new_stride"), (dict(budget=1 << 29, new_stride=1 << 29), -2, "too many")])
def test_evict_refusals(kw, code, word):
    lib = H.load()
    c = _cache(**{**dict(weights=0x5000), **kw})
    a = {**dict(new=0x6000, new_stride=2, budget=32, recent=8, kept=0x7000, left=0x8000), **kw}
    assert lib.attnres_cache_evict(ctypes.byref(c), a["new"], a["new_stride"], a["budget"], a["recent"], a["kept"], a["left"],
                                   None, 0, None) == code
    assert word in lib.attnres_last_error().decode()


@needs_lib
def test_evict_workspace():
    lib = H.load()
    short, long = _cache(weights=0x5000), _cache(weights=0x5000, table_pages=1 << 12, table_stride=1 << 12)
    assert lib.attnres_cache_evict_workspace_size(ctypes.byref(short), 32, 8) == 0
    n = lib.attnres_cache_evict_workspace_size(ctypes.byref(long), 32, 8)
    assert n > 0
    for ws, size in ((None, n), (0x100000, n - 1), (0x100010, n)):
        assert lib.attnres_cache_evict(ctypes.byref(long), 0x6000, 2, 32, 8, 0x7000, 0x8000, ws, size, None) == -4
        assert "workspace" in lib.attnres_last_error().decode()


def test_no_cpu_path():
    g = torch.Generator().manual_seed(0)
    c = Cache(g, torch.float32, 2, 8, 4, [3, 5], 8, device="cpu", weights=True)
    q = torch.randn((2, 4, 1, 8), generator=g)
    sin = cos = torch.ones((16, 4))
    for call in (lambda: ops.cached_attention(q, c.k, c.v, c.table, c.cached),
                 lambda: ops.qkv_norm_rotary_cached(torch.randn((2, 1, 64)), 4, sin, cos, c.k, c.v, c.table, c.cached),
                 lambda: ops.evict_cached_tokens(c.k, c.v, c.w, c.table, c.cached, c.table, 4, 1)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_reference_forms():
    """The 64-bit forms that the GPU tests go by, against attention written out."""
    g = torch.Generator().manual_seed(1)
    c = Cache(g, torch.float64, 2, 8, 4, [3, 5], 8, device="cpu")
    c.put(g, [5, 7])
    q = torch.randn((2, 4, 2, 8), generator=g, dtype=torch.float64)
    out = attend_ref(c, q.float(), [3, 5], [2, 2], 0.5)[0]
    for b, n in ((0, 5), (1, 7)):
        k, v = (c.get(t, b, n).repeat_interleave(2, 0) for t in (c.k, c.v))
        mask = torch.ones((2, n), dtype=torch.bool).tril(n - 2)
        e = torch.nn.functional.scaled_dot_product_attention(q[b].float().double(), k, v, attn_mask=mask, scale=0.5)
        assert torch.allclose(out[b], e, atol=1e-12)
    nan = float("nan")
    assert evict_ref([1.0, 3.0, 3.0, nan, 0.5, 9.0], 6, 3, 1) == [1, 2, 5]
    assert evict_ref([nan, nan, 0.0, -1.0], 4, 3, 0) == [0, 2, 3]
    assert evict_ref([1.0, 2.0], 2, 5, 1) == [0, 1]
