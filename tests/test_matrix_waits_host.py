"""CPU check of the attention kernels' generated code: no instruction reads a matrix product's result too soon.

The hardware does not wait for a product by itself: 8 issue slots (16 x 16 tiles of 16-bit operands) or 10 (fp32) have to lie
between it and what reads its registers, along every way through the code.  The compiler fills them, but has been seen to count only
the longer of two ways around a branch.
"""

import os
import re
import shutil
import subprocess

import pytest

import build

HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
needs_hipcc = pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
PKG = os.path.dirname(os.path.abspath(build.__file__))
MOST = 24  # slots after which any product has ended


def registers(operand):
    m = re.match(r"-?\|?([va])\[(\d+):(\d+)\]", operand) or re.match(r"-?\|?([va])(\d+)", operand)
    if not m:
        return frozenset()
    return frozenset((m[1], i) for i in range(int(m[2]), int(m[m.lastindex]) + 1))


def functions(text):
    """name -> [("label", name) or (operation, operands)] of every function of an assembly file"""
    out, code = {}, None
    for line in text.splitlines():
        line = line.split(";")[0].strip()
        if m := re.match(r"(_Z\w+):", line):
            code = out.setdefault(m[1], [])
        elif line.startswith(".Lfunc_end"):
            code = None
        elif code is not None and (m := re.match(r"(\.LBB\w+):", line)):
            code.append(("label", m[1]))
        elif code is not None and line and not line.startswith(".") and not line.endswith(":"):
            op, _, rest = line.partition(" ")
            code.append((op, [o.strip() for o in rest.split(",")] if rest else []))
    return out


def touched(op, operands):
    return frozenset().union(*(registers(o) for o in operands))


def shortest(code, at, labels):
    """Slots between the product at `at` and the first other instruction that reads or writes what is left of its result."""
    best, seen, ways = MOST, {}, [(at + 1, 0, registers(code[at][1][0]))]
    while ways:
        i, slots, result = ways.pop()
        if slots >= best or not result or i >= len(code) or seen.get((i, result), MOST) <= slots:
            continue
        seen[i, result] = slots
        op, operands = code[i]
        if op == "label":
            ways.append((i + 1, slots, result))
        elif op == "s_nop":
            ways.append((i + 1, slots + int(operands[0]) + 1, result))
        elif op == "s_branch":
            ways.append((labels[operands[0]], slots + 1, result))
        elif op.startswith("s_cbranch"):
            ways += [(labels[operands[0]], slots + 1, result), (i + 1, slots + 1, result)]
        elif op.startswith("v_mfma"):  # (products after one another wait by themselves)
            ways.append((i + 1, slots + 1, result - registers(operands[0])))
        elif touched(op, operands) & result:
            best = slots
        elif op != "s_endpgm":
            ways.append((i + 1, slots + 1, result))
    return best


def least(text):
    """operation -> fewest slots after it, over all functions"""
    out = {}
    for code in functions(text).values():
        labels = {name: i for i, (op, name) in enumerate(code) if op == "label"}
        for i, (op, _) in enumerate(code):
            if op.startswith("v_mfma"):
                out[op] = min(out.get(op, MOST), shortest(code, i, labels))
    return out


def test_the_walk_takes_the_short_way_around_a_branch():
    code = """_Zkernel:
\tv_mfma_f32_16x16x4_f32 a[64:67], v219, v65, a[64:67]
\ts_and_saveexec_b64 s[4:5], s[12:13]
\ts_cbranch_execz .LBB0_2
; %bb.1:
\tv_mul_lo_u32 v10, s41, v0
\ts_nop 9
.LBB0_2:  ; loop
\ts_or_b64 exec, exec, s[4:5]
\tv_accvgpr_read_b32 v8, a64
\ts_endpgm
.Lfunc_end0:
"""
    assert least(code) == {"v_mfma_f32_16x16x4_f32": 3}
    assert least(code.replace("\ts_and_save", "\ts_nop 15\n\ts_and_save")) == {"v_mfma_f32_16x16x4_f32": 19}
    assert least(code.replace("a64\n", "a68\n")) == {"v_mfma_f32_16x16x4_f32": MOST}


@needs_hipcc
def test_attention_kernels_wait_for_their_products(tmp_path):
    jobs = []
    for t in ("bf16", "f16", "f32"):
        out = str(tmp_path / (t + ".s"))
        src = os.path.join(PKG, "csrc", f"attnres_cache_attend_{t}.hip")
        jobs.append((t, out, subprocess.Popen([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-S",
                                               "--cuda-device-only", *build.DEVICE_FLAGS, src, "-o", out],
                                              stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)))
    for t, out, job in jobs:
        assert job.wait() == 0
        found = least(open(out).read())
        assert found and all(op.endswith("_" + t) for op in found), found
        assert min(found.values()) >= (10 if t == "f32" else 8), found
