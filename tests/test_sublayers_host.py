"""CPU checks of the sublayer operators (qkv_norm_rotary, swiglu_projection): the C ABI's exports, struct layouts and
refusals (nothing is launched), the Python functions' refusals, and the decoder's fused sublayers against the reference
model's golden vectors with the oracle standing in for the kernels."""

import ctypes
import os
import re
import subprocess

import pytest
import torch
from torch.nn import functional as F

import _attnres_hip as H
import attnres_decoder as AD
import attnres_ops as ops
from oracle import attnres_oracle as O
from decoder_util import OracleOps, build_from_case, lm_step, load_model_case, model_index

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "attnres_sublayers.h")
needs_lib = pytest.mark.skipif(not os.path.exists(H.LIB_PATH), reason="libattnres_hip.so not built")
STRUCTS = ((H.QkvRotaryDesc, "attnres_qkv_rotary_desc"), (H.SwigluDesc, "attnres_swiglu_desc"))


@needs_lib
def test_library_exports_every_declared_symbol():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(attnres_[a-z0-9_]+)\s*\(", text)))
    assert names == sorted(["attnres_qkv_rotary_forward", "attnres_qkv_rotary_backward", "attnres_swiglu_saved_size",
                            "attnres_swiglu_forward_workspace_size", "attnres_swiglu_backward_workspace_size",
                            "attnres_swiglu_forward", "attnres_swiglu_backward"])
    nm = subprocess.run(["nm", "-D", "--defined-only", H.LIB_PATH], capture_output=True, text=True).stdout
    for n in names:
        assert re.search(rf"\bT {n}\b", nm), n


def test_ctypes_structs_match_the_header(tmp_path):
    lines = [f'  printf("{n} sizeof %zu\\n", sizeof({n}));' for _, n in STRUCTS]
    lines += [f'  printf("{n} {f} %zu\\n", offsetof({n}, {f}));' for cls, n in STRUCTS for f, _ in cls._fields_]
    c, exe = tmp_path / "p.c", tmp_path / "p"
    c.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"attnres_sublayers.h\"\nint main(void) {\n" +
                 "\n".join(lines) + "\n  return 0;\n}\n")
    subprocess.run(["gcc", "-I", os.path.dirname(HEADER), str(c), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    lay = {tuple(line.split()[:2]): int(line.split()[2]) for line in out.strip().splitlines()}
    for cls, name in STRUCTS:
        assert ctypes.sizeof(cls) == lay[(name, "sizeof")]
        for f, _ in cls._fields_:
            assert getattr(cls, f).offset == lay[(name, f)], (name, f)


def _rotary(**kw):
    d = H.QkvRotaryDesc(dtype=1, table_dtype=0, batch=2, tokens=4, q_heads=4, kv_heads=2, head_dim=64, qk_norm=1,
                        norm_eps=1e-7, qkv=0x1000, batch_stride=4 * 512, token_stride=512, sin=0x2000, cos=0x3000,
                        table_rows=8, table_row_stride=32)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@needs_lib
@pytest.mark.parametrize("kw,code,word", [
    (dict(dtype=7), -1, "dtype"), (dict(table_dtype=2), -1, "table dtype"), (dict(batch=-1), -1, "batch"),
    (dict(q_heads=0), -1, "q_heads"), (dict(kv_heads=0), -1, "kv_heads"), (dict(head_dim=63), -1, "head_dim"),
    (dict(head_dim=0), -1, "head_dim"), (dict(head_dim=1026), -2, "head_dim"), (dict(qkv=0), -1, "NULL"),
    (dict(sin=0), -1, "NULL"), (dict(cos=0), -1, "NULL"), (dict(token_stride=-1), -1, "stride"),
    (dict(table_rows=0), -1, "table_rows"), (dict(table_row_stride=31), -1, "table_row_stride"),
    (dict(start=-1), -1, "outside"), (dict(start=5), -1, "outside"), (dict(table_rows=3), -1, "outside"),
    (dict(batch=1 << 40, tokens=1 << 30), -2, "tokens")])
def test_rotary_refusals(kw, code, word):
    lib = H.load()
    assert lib.attnres_qkv_rotary_forward(None, None, None, None) == -1
    d = _rotary(**kw)
    assert lib.attnres_qkv_rotary_forward(ctypes.byref(d), 0x4000, 0x5000, None) == code
    assert word in lib.attnres_last_error().decode()
    g, s = (ctypes.c_void_p * 3)(), (ctypes.c_int64 * 9)()
    assert lib.attnres_qkv_rotary_backward(ctypes.byref(d), g, s, 0x4000, None) == code


@needs_lib
def test_rotary_null_outputs_and_empty_calls():
    lib = H.load()
    d = _rotary()
    g, s = (ctypes.c_void_p * 3)(0x9000, None, None), (ctypes.c_int64 * 9)(-1)
    assert lib.attnres_qkv_rotary_forward(ctypes.byref(d), None, 0x5000, None) == -1
    assert lib.attnres_qkv_rotary_backward(ctypes.byref(d), None, s, 0x4000, None) == -1
    assert lib.attnres_qkv_rotary_backward(ctypes.byref(d), g, s, None, None) == -1
    assert lib.attnres_qkv_rotary_backward(ctypes.byref(d), g, s, 0x4000, None) == -1
    assert b"negative gradient stride" in lib.attnres_last_error()
    for kw in (dict(batch=0), dict(tokens=0)):
        d = _rotary(qkv=0, sin=0, cos=0, **kw)
        assert lib.attnres_qkv_rotary_forward(ctypes.byref(d), None, None, None) == 0
        assert lib.attnres_qkv_rotary_backward(ctypes.byref(d), g, s, None, None) == 0


def _swiglu(**kw):
    d = H.SwigluDesc(dtype=1, n_tok=100, dim=64, hidden=48, x=0x1000, x_row_stride=64, weight=0x2000,
                     weight_row_stride=64)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@needs_lib
@pytest.mark.parametrize("kw,code,word", [
    (dict(dtype=3), -1, "dtype"), (dict(n_tok=-1), -1, "n_tok"), (dict(dim=0), -1, "dim"), (dict(hidden=0), -1, "hidden"),
    (dict(n_tok=(1 << 22) + 1), -2, "32-bit"), (dict(dim=1 << 21), -2, "32-bit"), (dict(hidden=1 << 21), -2, "32-bit"),
    (dict(dim=1 << 16, hidden=1 << 16), -2, "32-bit"), (dict(x=0), -1, "NULL"), (dict(weight=0), -1, "NULL"),
    (dict(x_row_stride=-64), -1, "x_row_stride"), (dict(weight_row_stride=63), -1, "weight_row_stride")])
def test_swiglu_refusals(kw, code, word):
    lib = H.load()
    assert lib.attnres_swiglu_forward(None, None, None, None, 0, None) == -1
    d = _swiglu(**kw)
    assert lib.attnres_swiglu_forward(ctypes.byref(d), 0x4000, None, None, 0, None) == code
    assert word in lib.attnres_last_error().decode()
    assert lib.attnres_swiglu_backward(ctypes.byref(d), 0x4000, 48, 0x5000, 0x6000, 0x7000, None, 0, None) == code
    assert lib.attnres_swiglu_saved_size(ctypes.byref(d)) == 0
    assert lib.attnres_swiglu_backward_workspace_size(ctypes.byref(d), 1, 1) == 0


@needs_lib
def test_swiglu_sizes_workspaces_and_empty_calls():
    lib = H.load()
    # u and z of whole k steps (32 / 32 / 16 columns): 5, 6 and 8 bytes a pair
    for dtype, step, pair in ((1, 32, 5), (2, 32, 6), (0, 16, 8)):
        for n, hidden in ((1, 1), (100, 48), (7, 33)):
            d = _swiglu(dtype=dtype, n_tok=n, hidden=hidden)
            assert lib.attnres_swiglu_saved_size(ctypes.byref(d)) == n * -(-hidden // step) * step * pair
    d = _swiglu()
    need = lib.attnres_swiglu_backward_workspace_size(ctypes.byref(d), 1, 1)
    assert need >= 100 * 2 * 64 * 2
    args = (ctypes.byref(d), 0x4000, 48, 0x5000, 0x6000, 0x7000)
    assert lib.attnres_swiglu_backward(*args, None, need, None) == -4
    assert lib.attnres_swiglu_backward(*args, 0x10000, need - 1, None) == -4
    assert lib.attnres_swiglu_backward(*args, 0x10010, need, None) == -4
    assert lib.attnres_swiglu_forward(ctypes.byref(d), None, None, None, 0, None) == -1
    assert lib.attnres_swiglu_forward(ctypes.byref(d), 0x4000, 0x5008, None, 0, None) == -1
    assert lib.attnres_swiglu_backward(ctypes.byref(d), 0x4000, -1, 0x5000, 0x6000, 0x7000, 0x10000, need, None) == -1
    assert lib.attnres_swiglu_backward(ctypes.byref(d), None, 48, 0x5000, 0x6000, 0x7000, 0x10000, need, None) == -1
    # an operand that 16-byte loads cannot address is copied: there has to be room
    odd = _swiglu(x=0x1002)
    assert lib.attnres_swiglu_forward_workspace_size(ctypes.byref(odd)) >= 100 * 64 * 2
    assert lib.attnres_swiglu_forward(ctypes.byref(odd), 0x4000, None, None, 0, None) == -4
    assert lib.attnres_swiglu_forward(ctypes.byref(_swiglu(n_tok=0, x=0, weight=0)), None, None, None, 0, None) == 0
    # nothing asked for: nothing done
    assert lib.attnres_swiglu_backward(ctypes.byref(d), 0x4000, 48, 0x5000, None, None, None, 0, None) == 0


def test_python_refusals():
    sin = cos = torch.zeros(8, 4)
    qkv = torch.zeros(1, 4, 6 * 8)
    bad = [
        (lambda: ops.qkv_norm_rotary(qkv[0], 2, sin, cos), "must be"),
        (lambda: ops.qkv_norm_rotary(qkv.double(), 2, sin, cos), "dtype"),
        (lambda: ops.qkv_norm_rotary(qkv, 0, sin, cos), "num_heads"),
        (lambda: ops.qkv_norm_rotary(qkv, 2, sin, cos, num_kv_heads=0), "num_kv_heads"),
        (lambda: ops.qkv_norm_rotary(qkv, 5, sin, cos), "heads of an even width"),
        (lambda: ops.qkv_norm_rotary(qkv[..., :18], 2, sin, cos), "heads of an even width"),
        (lambda: ops.qkv_norm_rotary(torch.zeros(1, 1, 3 * 1026), 1, sin, cos), "above 1024"),
        (lambda: ops.qkv_norm_rotary(qkv, 2, sin[:, :3], cos), "sin must be"),
        (lambda: ops.qkv_norm_rotary(qkv, 2, sin, cos[0]), "cos must be"),
        (lambda: ops.qkv_norm_rotary(qkv, 2, sin, cos[:4]), "differ in shape"),
        (lambda: ops.qkv_norm_rotary(qkv, 2, torch.zeros(2, 8, 4), torch.zeros(2, 8, 4)), "sin must be"),
        (lambda: ops.qkv_norm_rotary(qkv, 2, sin.clone().requires_grad_(True), cos), "no gradient"),
        (lambda: ops.qkv_norm_rotary(qkv, 2, sin.long(), cos.long()), "floating-point"),
        (lambda: ops.qkv_norm_rotary(qkv, 2, sin, cos), "ROCm GPU"),
        (lambda: ops.swiglu_projection(torch.zeros(()), torch.zeros(4, 1)), "x must be"),
        (lambda: ops.swiglu_projection(torch.zeros(2, 8).double(), torch.zeros(4, 8)), "dtype"),
        (lambda: ops.swiglu_projection(torch.zeros(2, 8), torch.zeros(4, 7)), "weight must be"),
        (lambda: ops.swiglu_projection(torch.zeros(2, 8), torch.zeros(3, 8)), "weight must be"),
        (lambda: ops.swiglu_projection(torch.zeros(2, 8), torch.zeros(0, 8)), "weight must be"),
        (lambda: ops.swiglu_projection(torch.zeros(2, 0), torch.zeros(4, 0)), "weight must be"),
        (lambda: ops.swiglu_projection(torch.zeros(2, 8), torch.zeros(4, 8).long()), "floating-point"),
        (lambda: ops.swiglu_projection(torch.zeros(2, 8), torch.zeros(4, 8)), "ROCm GPU"),
    ]
    for f, word in bad:
        with pytest.raises(RuntimeError, match=word):
            f()


class _FusedOracle(OracleOps):
    qkv_norm_rotary = staticmethod(O.qkv_norm_rotary_ref)
    swiglu_projection = staticmethod(O.swiglu_projection_ref)


@pytest.mark.parametrize("name", sorted(model_index()))
def test_decoder_with_fused_sublayers_matches_reference_model(name):
    """The oracle's functions compose the reference's own ops, so the decoder that calls them in the fused sublayers'
    place reproduces the golden hidden state, loss and gradients bit for bit: pins what the kernels stand for."""
    t, meta = load_model_case(name)
    model = build_from_case(t, meta, _FusedOracle, fuse_qkv_rotary=True, fuse_swiglu=True)
    hidden, loss = lm_step(model, t["idx"], t["targets"])
    assert torch.equal(hidden, t["hidden"]) and torch.equal(loss.reshape(1), t["loss"])
    for pname, p in model.named_parameters():
        assert torch.equal(p.grad, t[f"grad.{pname}"]), pname


def test_fused_sublayers_are_off_by_default():
    c = AD.DecoderConfig()
    assert not c.fuse_qkv_rotary and not c.fuse_swiglu
    assert AD.Decoder(AD.DecoderConfig(n_layer=1, n_head=1, n_embd=8, vocab_size=8, use_attnres=False)).ops is None
    cfg = AD.DecoderConfig(n_layer=1, n_head=1, n_embd=8, vocab_size=8, use_attnres=False, fuse_swiglu=True)
    assert AD.Decoder(cfg).ops is ops


def test_oracle_positions_and_grouped_heads():
    """The parts of the oracle that the reference does not have: positions by index, and fewer key / value heads."""
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(2, 5, (4 + 2 * 2) * 6, generator=g, dtype=torch.float64)
    a = torch.outer(torch.arange(9, dtype=torch.float64), torch.rand(3, generator=g, dtype=torch.float64))
    at = torch.randint(0, 9, (2, 5), generator=g)
    q, k, v = O.qkv_norm_rotary_ref(qkv, 4, a.sin(), a.cos(), at, 2)
    heads = qkv.view(2, 5, 8, 6).transpose(1, 2)
    for b in range(2):
        for h in range(8):
            for t in range(5):
                x = heads[b, h, t]
                if h >= 6:
                    assert torch.equal(v[b, h - 6, t], x)
                    continue
                n = F.rms_norm(x, (6,))
                z = torch.view_as_complex(n.view(3, 2)) * torch.polar(torch.ones(3, dtype=torch.float64), a[at[b, t]])
                got = q[b, h, t] if h < 4 else k[b, h - 4, t]
                assert torch.allclose(got, torch.view_as_real(z).flatten(), rtol=0, atol=1e-14)
