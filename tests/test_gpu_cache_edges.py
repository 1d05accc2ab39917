"""The paged cache's operators at the edges of what they are given: counts and positions that 32 bits do not hold, pages that
some rows read and others do not, several new tokens whose rows are joined from pieces."""

import pytest
import torch

import attnres_ops as ops
from cache_util import Cache, assert_within, attend_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
I32 = dict(dtype=torch.int32, device=DEV)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def same(a, b):
    """Bit for bit, and NaN in the same places."""
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0.0), b.nan_to_num(0.0))


def queries(g, B, H, T, Dh, dtype):
    return (torch.randn((B, H, T, Dh), generator=g) * 2.0).to(dtype).to(DEV)


def test_positions_and_counts_of_64_bits_below_zero():
    """Rows below zero are outside the tables however far: no later token of the call takes an early row by them."""
    H, K, Dh, T, rows = 4, 2, 64, 9, 40
    g = gen(1)
    c = Cache(g, torch.bfloat16, K, Dh, 16, [3, 3, 3, 3], 32, fill=0.125)
    qkv = torch.randn((4, T, (H + 2 * K) * Dh), generator=g).to(torch.bfloat16).to(DEV)
    angle = torch.rand((rows, Dh // 2), generator=g)
    sin, cos = angle.sin().to(DEV), angle.cos().to(DEV)

    def call(cached, positions=None):
        c.k.fill_(0.125), c.v.fill_(0.125)
        out = ops.qkv_norm_rotary_cached(qkv, H, sin, cos, c.k, c.v, c.table, cached, positions=positions, return_heads=True)
        return [*out[:2], c.k.clone(), c.v.clone()]

    far64 = torch.tensor([-5, -2 ** 40, 2 ** 40, 2], device=DEV)
    far32 = torch.tensor([-5, -2 ** 31, 2 ** 31 - 1, 2], **I32)
    want = call(c.cached, far32)
    for a, b in zip(call(c.cached, far64), want):
        assert same(a, b)
    for t in want[:2]:
        bad = t.isnan().all(-1).all(1)
        assert bad.tolist() == [[True] * 5 + [False] * 4, [True] * T, [True] * T, [False] * T]
    # row t - 5 of the tables, as the same call from row 0 on takes it
    zero = torch.zeros((4,), **I32)
    shifted = ops.qkv_norm_rotary_cached(qkv[:, 5:], H, sin, cos, c.k, c.v, c.table, c.cached, positions=zero)
    assert torch.equal(want[0][0, :, 5:], shifted[0])
    # counts, which positions come from unless given
    for a, b in zip(call(torch.tensor([-5, -2 ** 40, 2 ** 40, 2], device=DEV)), call(far32)):
        assert same(a, b)
    assert bool((call(far64)[2][c.table[:3].long()] == 0.125).all()), "nothing is written for counts that cannot be"
    q = queries(g, 4, H, 2, Dh, torch.bfloat16)
    c.k.fill_(0.125), c.v.fill_(0.125)
    a, b = (ops.cached_attention(q, c.k, c.v, c.table, n) for n in (far64, far32))
    assert same(a, b) and a.isnan().all(-1).all(-1).all(-1).tolist() == [True, True, True, False]
    # (a table that 32 bits cannot name all rows of, without its memory: the call is refused before it is looked at)
    huge = sin[:1].expand(2 ** 31, -1)
    with pytest.raises(RuntimeError, match="positions of 64 bits"):
        ops.qkv_norm_rotary_cached(qkv, H, huge, huge, c.k, c.v, c.table, c.cached, positions=far64)
