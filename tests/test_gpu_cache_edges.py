"""The paged cache's operators at the edges of what they are given: counts and positions that 32 bits do not hold, pages that
some rows read and others do not, several new tokens whose rows are joined from pieces."""

import ctypes

import pytest
import torch

import _attnres_hip as lib
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


def widen(c, rows):
    """Columns of the table that no token is in, as many as make it a call of many bytes: blocks of 32 rows."""
    columns = -(-(256 << 20) // (c.B * c.K * -(-rows // 16) * 2 * c.Dh * c.k.element_size() * c.S)) + 1
    more = torch.full((c.B, max(0, columns - c.table.size(1))), -7, **I32)
    c.table = torch.cat([c.table, more], 1)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype,Dh", [("bf16", 64), ("fp16", 128), ("fp32", 40)])
@pytest.mark.parametrize("S,T", [(16, 2), (16, 20), (32, 5), (24, 2), (24, 20), (7, 9), (1, 3)])
def test_rows_that_do_not_read_a_missing_page(S, T, dtype, Dh, wide):
    """Rows up to the last token of a page, the next one missing: those that read it are NaN, the others as if it were there."""
    H, K = 4, 2
    cached = [max(0, 2 * S - 1 - T // 2), 5 * S - 1, 3]
    g = gen(S * T)
    c = Cache(g, DT[dtype], K, Dh, S, cached, max(cached) + T + S)
    c.put(g, [n + T for n in cached])
    q = queries(g, 3, H, T, Dh, DT[dtype])
    if wide:
        widen(c, 2 * T)
    e, bound, _ = attend_ref(c, q, cached, [T] * 3, Dh ** -0.5)
    good = ops.cached_attention(q, c.k, c.v, c.table, c.cached)
    assert_within(good, e, bound, "all pages there")
    first = [2 * S, 5 * S]  # tokens of the missing pages
    c.table[0, 2], c.table[1, 5] = -1, c.k.size(0)
    o = ops.cached_attention(q, c.k, c.v, c.table, c.cached)
    for b in range(2):
        for t in range(T):
            if cached[b] + t >= first[b]:
                assert bool(o[b, :, t].isnan().all()), (b, t)
            else:
                assert_within(o[b, :, t], e[b, :, t], bound[b, :, t], f"sequence {b}, row {t}")
    assert cached[0] < first[0] and cached[1] < first[1] <= cached[1] + T - 1
    assert torch.equal(o[2], good[2])


def workspace(c, q):
    """Workspace bytes of a call, and what pieces of 256 workgroups' blocks of 16 rows take at most."""
    d = lib.CacheAttendDesc()
    d.q_heads, d.tokens, d.scale, d.q = q.size(1), q.size(2), 0.125, q.data_ptr()
    n = lib.load().attnres_cache_attend_workspace_size(
        ctypes.byref(lib.cache_desc(c.k, c.v, None, c.table, c.cached, None)), ctypes.byref(d))
    tile = 64 if c.Dh <= 64 else 128 if c.Dh <= 128 else 256
    return n, 2 * 256 * 16 * (tile + 2) * 4


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,H,K,Dh,S,layout", [
    (7, 16, 4, 64, 32, "dense"), (4, 4, 4, 40, 24, "dense"), (9, 6, 2, 17, 7, "dense"), (20, 2, 1, 96, 20, "dense"),
    (5, 8, 2, 96, 16, "dense"), (33, 2, 2, 64, 16, "tokens"), (3, 20, 2, 40, 24, "odd"), (6, 3, 1, 200, 20, "layer"),
    (2, 1, 1, 256, 64, "dense"), (17, 2, 2, 62, 48, "dense")])
def test_several_new_tokens_of_split_rows(dtype, T, H, K, Dh, S, layout):
    """Tables so long that rows are read in pieces and joined, too short for blocks of 32 rows; padding among the new tokens."""
    cached = [0, 5, 700, 2600, 131]
    fresh = [T, 1, T - 1, T, 0]
    g = gen(T * Dh + S)
    c = Cache(g, DT[dtype], K, Dh, S, cached, max(cached) + T, layout)
    c.put(g, [n + f for n, f in zip(cached, fresh)])
    # (columns that no token is in, up to 1 MiB of keys and values a head and a little more)
    need = -(-((1 << 20) + 4096) // (2 * Dh * c.k.element_size() * S))
    more = torch.full((c.B, max(0, need - c.table.size(1))), 10 ** 9, **I32)
    c.table = torch.cat([c.table, more], 1)
    q = queries(g, c.B, H, T, Dh, DT[dtype])
    n, most = workspace(c, q)
    assert 0 < n <= most, "pieces, of blocks of 16 rows"
    f = torch.tensor(fresh, **I32)
    e, bound, _ = attend_ref(c, q, cached, fresh, Dh ** -0.5)
    o = ops.cached_attention(q, c.k, c.v, c.table, c.cached, fresh=f)
    assert_within(o, e, bound, "out")
    for b, k in enumerate(fresh):
        assert not bool(o[b, :, k:].any()), "rows that no sequence has are zeros"
    assert torch.equal(ops.cached_attention(q, c.k, c.v, c.table, c.cached, fresh=f), o)


def test_the_most_heads_that_a_call_takes():
    """3 x 715827882 heads, 2 below 2^31, a wave each (rows that start anywhere): the grid's two dimensions end behind 2^31
    waves, and those have no head."""
    T, Dh = (2 ** 31 - 1) // 3, 2
    flat = torch.zeros((T * 3 * Dh + 1,), dtype=torch.float16, device=DEV)
    qkv = flat[1:].view(1, T, 3 * Dh)
    qkv[:, :5] = torch.randn((1, 5, 3 * Dh), generator=gen(2)).to(torch.float16).to(DEV)
    qkv[:, 5:8] = 1.0  # (padding: in no query, no page)
    qkv[:, -3:] = 1.0
    angle = torch.rand((8, Dh // 2), generator=gen(3))
    sin, cos = angle.sin().to(DEV), angle.cos().to(DEV)
    c = Cache(gen(4), torch.float16, 1, Dh, 4, [0], 8, fill=0.125)
    q = ops.qkv_norm_rotary_cached(qkv, 1, sin, cos, c.k, c.v, c.table, c.cached, fresh=torch.tensor([5], **I32))
    k, v = c.k.clone(), c.v.clone()
    c.k.fill_(0.125), c.v.fill_(0.125)
    want = ops.qkv_norm_rotary_cached(qkv[:, :5], 1, sin, cos, c.k, c.v, c.table, c.cached)
    assert torch.equal(q[:, :, :5], want) and torch.equal(k, c.k) and torch.equal(v, c.v)
    assert not bool(q[:, :, 5:].any())


@pytest.mark.parametrize("gap", [5.0, 26.0, 40.0, 60.0])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T", [1, 3])
def test_an_infinite_value_of_a_small_weight(dtype, gap, T):
    """exp(-gap) times an infinite value is infinite, not NaN, however much smaller than a 16-bit term it is; the other columns
    and the rows before it are as ever."""
    g = gen(int(gap))
    cached = [130, 150]  # (tokens 0 .. 31 and 128 .. 159 are one wave's)
    c = Cache(g, DT[dtype], 1, 64, 16, cached, 160)
    c.put(g, [n + T for n in cached], std=0.125)
    q = torch.zeros((2, 2, T, 64), dtype=DT[dtype], device=DEV)
    q[..., 0] = 8.0  # scores are the keys' first values
    for b, n in enumerate(cached):
        page, slot = c.where(b, n + T)
        c.k[page, 0, slot, 0] = 0.0
        c.k[page[20], 0, slot[20], 0] = gap  # one token has the largest score, all others are `gap` below
        last = n + T - 1                      # (the last new token: rows before it do not see it)
        c.v[page[last], 0, slot[last], 7] = float("inf")
        c.v[page[27], 0, slot[27], 9] = -float("inf")
    e, bound, _ = attend_ref(c, q, cached, [T, T], 0.125)
    o = ops.cached_attention(q, c.k, c.v, c.table, c.cached, scale=0.125)
    assert bool((o[:, :, T - 1, 7] == float("inf")).all()) and bool((o[..., 9] == -float("inf")).all())
    fine = torch.isfinite(e)
    assert int((~fine).sum()) == 2 * 2 * (T + 1)
    assert_within(o[fine], e[fine], bound[fine], "finite")
