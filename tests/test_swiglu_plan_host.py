"""Host-side planning of the gated projections' backward through the C ABI (nothing is launched): a product whose gradient
is not asked for neither refuses a call nor asks for memory."""

import ctypes
import os

import pytest

import _attnres_hip as H

pytestmark = pytest.mark.skipif(not os.path.exists(H.LIB_PATH), reason="libattnres_hip.so not built")

# 2^22 tokens of 2^18 values: the input's gradient has 2^24 tiles of 256 x 256, one too many for a launch
WIDE = dict(dtype=1, n_tok=1 << 22, dim=1 << 18, hidden=32, x=0x1000, x_row_stride=0, weight=0x2000,
            weight_row_stride=1 << 18)


def _backward(d, dx, dw, workspace_bytes):
    # (too small a workspace: refused before anything could be launched)
    return H.load().attnres_swiglu_backward(ctypes.byref(d), 0x10000, 32, 0x20000, dx, dw, 0x30000, workspace_bytes, None)


def test_a_gradient_that_is_not_wanted_refuses_nothing():
    lib, d = H.load(), H.SwigluDesc(**WIDE)
    assert _backward(d, 0x40000, 0x50000, 0) == -2
    assert b"too many tiles" in lib.attnres_last_error()
    assert _backward(d, 0x40000, None, 0) == -2
    assert _backward(d, None, 0x50000, 0) == -4  # (the weight's gradient alone: only the workspace is missing)


@pytest.mark.parametrize("shape", [(100, 64, 48), (2031, 500, 1363), (16384, 768, 2048)])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_workspace_asked_for_is_workspace_needed(shape, dtype):
    lib = H.load()
    n, dim, hidden = shape
    for shift in (0, 2):  # operands where they are, copied
        d = H.SwigluDesc(dtype=dtype, n_tok=n, dim=dim, hidden=hidden, x=0x1000 + shift, x_row_stride=dim,
                         weight=0x2000 + shift, weight_row_stride=dim)
        both = lib.attnres_swiglu_backward_workspace_size(ctypes.byref(d), 1, 1)
        for dx, dw in ((0x40000, None), (None, 0x50000), (0x40000, 0x50000)):
            need = lib.attnres_swiglu_backward_workspace_size(ctypes.byref(d), dx is not None, dw is not None)
            assert 0 < need <= both
            assert _backward(d, dx, dw, need - 1) == -4
            assert f"{need} bytes needed".encode() in lib.attnres_last_error()
