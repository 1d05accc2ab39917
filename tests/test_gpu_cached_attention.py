"""cached_attention against its definition in 64 bits: types, group sizes, head widths, page sizes and layouts, lengths from
one token on, padded batches, several new tokens, received weights, bad tables, graphs and streams."""

import math

import pytest
import torch

import attnres_ops as ops
from cache_util import Cache, assert_within, attend_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def queries(g, B, H, T, Dh, dtype, std=2.0):
    return (torch.randn((B, H, T, Dh), generator=g) * std).to(dtype).to(DEV)


def build(seed, dtype, H, K, Dh, S, cached, T=1, layout="dense", fresh=None, weights=False, room=None):
    g = gen(seed)
    fresh = [T] * len(cached) if fresh is None else fresh
    c = Cache(g, DT[dtype], K, Dh, S, cached, max(cached) + T if room is None else room, layout, weights=weights)
    c.put(g, [n + f for n, f in zip(cached, fresh)])
    return c, queries(g, len(cached), H, T, Dh, DT[dtype]), fresh


def check(c, q, cached, fresh, pass_fresh=False, scale=None, **kw):
    f = torch.tensor(fresh, dtype=torch.int32, device=DEV) if pass_fresh else None
    o = ops.cached_attention(q, c.k, c.v, c.table, c.cached, fresh=f, scale=scale, **kw)
    e, bound, ps = attend_ref(c, q, cached, fresh, q.size(-1) ** -0.5 if scale is None else scale)
    assert o.shape == q.shape and o.dtype == q.dtype
    assert_within(o, e, bound, "out")
    return o, ps


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("H,K,Dh,S", [
    (1, 1, 64, 64), (12, 12, 64, 16), (8, 2, 128, 32), (16, 1, 64, 64), (20, 1, 96, 48), (6, 2, 256, 128), (3, 3, 40, 24),
    (4, 4, 32, 1), (2, 1, 20, 5), (5, 5, 17, 7), (34, 2, 80, 20), (4, 2, 8, 256), (2, 2, 200, 100),
    (4, 2, 148, 64), (2, 1, 134, 16), (3, 1, 62, 32), (2, 2, 36, 24), (8, 1, 196, 32), (2, 1, 129, 16), (6, 2, 100, 48),
    (2, 2, 1, 16), (3, 1, 254, 20)])
def test_lengths_and_shapes(dtype, H, K, Dh, S):
    cached = [0, 1, 30, 31, 32, 63, 64, 65, 127, 128, 129, 300]
    c, q, fresh = build(H * 131 + Dh, dtype, H, K, Dh, S, cached)
    check(c, q, cached, fresh)


@pytest.mark.parametrize("dtype,H,K,Dh,S,cached", [
    ("bf16", 4, 2, 64, 64, [5000]), ("bf16", 8, 1, 128, 16, [3, 9000, 40]), ("fp32", 2, 2, 64, 24, [4097, 0]),
    ("fp16", 2, 1, 256, 40, [2047, 2048, 2049]), ("bf16", 1, 1, 64, 64, [40000])])
def test_long(dtype, H, K, Dh, S, cached):
    c, q, fresh = build(7, dtype, H, K, Dh, S, cached)
    check(c, q, cached, fresh)


@pytest.mark.parametrize("batch", [65, 300])
def test_many_sequences(batch):
    g = gen(batch)
    cached = torch.randint(0, 70, (batch,), generator=g).tolist()
    c, q, fresh = build(batch, "bf16", 4, 2, 32, 16, cached)
    check(c, q, cached, fresh)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("layout", ["tokens", "layer", "odd"])
@pytest.mark.parametrize("Dh,S", [(64, 32), (40, 9), (128, 16)])
def test_layouts(dtype, layout, Dh, S):
    cached = [0, 17, 200, 150]
    c, q, fresh = build(11, dtype, 6, 3, Dh, S, cached, layout=layout)
    check(c, q, cached, fresh)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,H,K,Dh,S", [(2, 4, 4, 64, 64), (7, 16, 4, 64, 32), (16, 3, 3, 40, 24), (33, 8, 2, 128, 16), (5, 40, 2, 32, 64)])
def test_several_new_tokens(dtype, T, H, K, Dh, S):
    cached = [0, 1, 29, 100, 260]
    c, q, fresh = build(T, dtype, H, K, Dh, S, cached, T=T)
    check(c, q, cached, fresh)


@pytest.mark.parametrize("dtype,T,H,K,Dh,S", [("bf16", 200, 4, 2, 64, 64), ("fp16", 150, 3, 1, 96, 20), ("fp32", 140, 2, 2, 32, 16)])
def test_a_prompt_after_cached_tokens(dtype, T, H, K, Dh, S):
    """Rows of far apart tokens, each block of them with its own last one."""
    cached = [0, 90, 517]
    fresh = [T, T - 1, T // 3]
    c, q, _ = build(T, dtype, H, K, Dh, S, cached, T=T, fresh=fresh)
    check(c, q, cached, fresh, pass_fresh=True)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,cached", [(1, [600, 3]), (1, [9000, 2]), (5, [600, 3]), (20, [5000])])
def test_the_largest_values(dtype, T, cached):
    """Sums of weights times values that only their mean keeps finite."""
    c, q, fresh = build(59, dtype, 4, 2, 64, 16, cached, T=T)
    for b, n in enumerate(cached):
        page, slot = c.where(b, n + T)
        sign = torch.randint(0, 2, (n + T, 2, 64), generator=gen(b)) * 2.0 - 1.0
        sign[:, :, :32] = 1.0
        c.v[page, :, slot] = (sign * 0.9 * torch.finfo(DT[dtype]).max).to(DT[dtype]).to(DEV)
    o, _ = check(c, q, cached, fresh)
    assert bool(torch.isfinite(o).all())


@pytest.mark.parametrize("T", [17, 40])
def test_values_that_are_not_finite_in_a_prompt(T):
    """Each row takes what its own token sees of them, in blocks of rows and tiles of tokens that do not end together."""
    cached = [70]
    c, q, fresh = build(T, "bf16", 2, 1, 64, 16, cached, T=T)
    page, slot = c.where(0, 70 + T)
    for bad in (0, 9, T - 2):
        c.v[page[70 + bad], 0, slot[70 + bad], bad] = float("inf")
    o = ops.cached_attention(q, c.k, c.v, c.table, c.cached)
    e, bound, _ = attend_ref(c, q, cached, fresh, 64 ** -0.5)
    for bad in (0, 9, T - 2):
        assert bool((o[0, :, bad:, bad] == math.inf).all()) and bool(torch.isfinite(o[0, :, :bad, bad]).all())
    fine = torch.isfinite(e)
    assert torch.equal(torch.isfinite(o), fine)
    assert_within(o[fine], e[fine], bound[fine], "finite")


@pytest.mark.parametrize("T", [1, 4, 20])
def test_padded_batch(T):
    cached = [0, 0, 50, 131, 7]
    fresh = [0, T, T // 2, 0, T]
    c, q, _ = build(T, "bf16", 4, 2, 64, 16, cached, T=T, fresh=fresh)
    o, _ = check(c, q, cached, fresh, pass_fresh=True)
    for b, f in enumerate(fresh):
        assert not bool(o[b, :, f:].any()), "rows that no sequence has are zeros"
    # (an empty sequence among them saw nothing at all)
    assert bool(torch.isfinite(o).all())


@pytest.mark.parametrize("T", [2, 18])
def test_later_tokens_do_not_reach_earlier_rows(T):
    """A draft's own value of NaN and infinities, and a NaN key, show in the rows that see it and in no other."""
    cached = [3, 62]
    c, q, fresh = build(3, "bf16", 4, 2, 64, 16, cached, T=T)
    bad = T // 2
    for b, n in enumerate(cached):
        page, slot = c.where(b, n + T)
        c.v[page[n + bad], 0, slot[n + bad], 5] = float("nan")
        c.v[page[n + bad], 0, slot[n + bad], 6] = float("inf")
        c.k[page[n + bad], 1, slot[n + bad], 7] = float("nan")
    o = ops.cached_attention(q, c.k, c.v, c.table, c.cached)
    e, bound, _ = attend_ref(c, q, cached, fresh, 64 ** -0.5)
    assert_within(o[:, :, :bad], e[:, :, :bad], bound[:, :, :bad], "rows before")
    later = o[:, :2, bad:]  # of key / value head 0
    assert bool(later[..., 5].isnan().all()) and bool((later[..., 6] == math.inf).all())
    keep = [d for d in range(64) if d not in (5, 6)]
    assert_within(later[..., keep], e[:, :2, bad:][..., keep], bound[:, :2, bad:][..., keep], "other columns")
    assert bool(o[:, 2:, bad:].isnan().all())


def test_scores_of_all_sizes():
    """Huge, equal and infinite scores: a softmax that is one token's, the mean, and NaN where there is no softmax."""
    cached = [100, 100, 100, 100]
    c, q, fresh = build(5, "fp32", 2, 2, 64, 16, cached)
    q[1] = 0.0
    o, _ = check(c, q, cached, fresh, scale=40.0)
    page, slot = c.where(2, 101)
    c.k[page, :, slot, 0] = -math.inf   # every score -inf: no softmax
    q[2, :, :, 0] = 1.0
    page, slot = c.where(3, 101)
    c.k[page[:40], :, slot[:40], 0] = -math.inf   # the first forty see nothing
    q[3, :, :, 0] = 1.0
    o = ops.cached_attention(q, c.k, c.v, c.table, c.cached)
    e, bound, _ = attend_ref(c, q, cached, fresh, 64 ** -0.5)
    assert bool(o[2].isnan().all())
    # (infinite products are in no bound: the others' alone)
    bound[3] = 1e-4
    assert_within(o[[0, 1, 3]], e[[0, 1, 3]], bound[[0, 1, 3]], "finite rows")


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("H,K,Dh,S,cached", [
    (4, 4, 64, 64, [0, 31, 200]), (16, 2, 128, 16, [300, 1000, 5]), (40, 2, 32, 24, [77, 0]), (3, 3, 17, 7, [50, 129])])
@pytest.mark.parametrize("decay", [0.0, 1.0, 0.75])
def test_received_weights(dtype, H, K, Dh, S, cached, decay):
    c, q, fresh = build(9, dtype, H, K, Dh, S, cached, weights=True)
    if decay == 0.0:
        c.w.fill_(float("nan"))  # what a page's last user left is not read
    before = c.w.clone()
    _, ps = check(c, q, cached, fresh, weights=c.w, decay=decay)
    e, bound = before.double(), torch.zeros_like(before, dtype=torch.float64)
    for b, n in enumerate(cached):
        page, slot = c.where(b, n + 1)
        for h in range(K):
            rows = [ps[b, i, 0] for i in range(h * (H // K), (h + 1) * (H // K))]
            got = sum(p for p, _ in rows)
            old = before[page, h, slot].double()
            e[page, h, slot] = got + (decay * old if decay else 0.0)
            # each weight's share, the group's fp32 sum, the product with the decay and the last sum
            bound[page, h, slot] = got * (rows[0][1] + max(s for _, s in rows) + (len(rows) + 4) * 2.0 ** -24) + \
                (3 * 2.0 ** -24 * old if decay else 0.0) + 1e-37
    touched = bound > 0
    assert_within(c.w[touched], e[touched], bound[touched], "weights")
    assert torch.equal(c.w[~touched].nan_to_num(7.0), before[~touched].nan_to_num(7.0)), "other slots are left as they were"


@pytest.mark.parametrize("dtype,H,K,Dh,S,cached", [
    ("bf16", 300, 1, 32, 16, [200, 3]), ("fp32", 520, 2, 16, 20, [90]), ("bf16", 4, 2, 64, 64, [6000, 100, 0]),
    ("fp16", 2, 2, 128, 16, [131, 0, 5, 260] * 18)])
def test_received_weights_of_many_heads_tokens_and_sequences(dtype, H, K, Dh, S, cached):
    test_received_weights(dtype, H, K, Dh, S, cached, 0.5)


def widen(c, rows):
    """Columns of the table that no token is in, as many as make it a call of many bytes: blocks of 32 rows."""
    columns = -(-(256 << 20) // (c.B * c.K * -(-rows // 16) * 2 * c.Dh * c.k.element_size() * c.S)) + 1
    more = torch.full((c.B, max(0, columns - c.table.size(1))), -7, dtype=torch.int32, device=DEV)
    c.table = torch.cat([c.table, more], 1)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,H,K,Dh,S", [(5, 8, 2, 64, 64), (17, 1, 1, 128, 16), (9, 8, 2, 128, 32), (6, 6, 1, 256, 64), (40, 2, 2, 48, 16),
                                        (3, 44, 2, 80, 128), (2, 20, 1, 200, 32)])
def test_blocks_of_many_rows(dtype, T, H, K, Dh, S):
    cached = [0, 1, 30, 127, 128, 333, 900]
    fresh = [T, T, T - 1, 0, T, T, 1]
    c, q, _ = build(T * Dh, dtype, H, K, Dh, S, cached, T=T, fresh=fresh)
    widen(c, T * (H // K))
    check(c, q, cached, fresh, pass_fresh=True)
    check(c, q.flip(-1), cached, fresh, pass_fresh=True, scale=-0.4)


@pytest.mark.parametrize("dtype,T,H,K,Dh,batch", [("bf16", 150, 8, 2, 64, 2), ("fp32", 9, 4, 2, 16, 70)])
def test_more_rows_than_workgroups_that_join(dtype, T, H, K, Dh, batch):
    g = gen(T)
    cached = torch.randint(0, 400, (batch,), generator=g).tolist()
    fresh = [T, *torch.randint(0, T + 1, (batch - 1,), generator=g).tolist()]
    assert batch * H * T > 2048
    c, q, _ = build(T, dtype, H, K, Dh, 16, cached, T=T, fresh=fresh)
    widen(c, T * (H // K))
    check(c, q, cached, fresh, pass_fresh=True)


@pytest.mark.parametrize("T", [17, 40])
def test_what_is_not_finite_in_blocks_of_many_rows(T):
    cached = [70, 300]
    c, q, fresh = build(T, "bf16", 4, 2, 64, 16, cached, T=T)
    for b, n in enumerate(cached):
        page, slot = c.where(b, n + T)
        for bad in (0, 9, T - 2):
            c.v[page[n + bad], 0, slot[n + bad], bad] = -float("inf")
            c.v[page[n + bad], 1, slot[n + bad], bad] = torch.finfo(torch.bfloat16).max
    widen(c, 2 * T)
    c.table[0, (70 + T) // 16 + 1:] = 10 ** 9
    o = ops.cached_attention(q, c.k, c.v, c.table, c.cached)
    e, bound, _ = attend_ref(c, q, cached, fresh, 64 ** -0.5)
    fine = torch.isfinite(e)
    assert torch.equal(torch.isfinite(o), fine) and bool((o[~fine] == -math.inf).all())
    assert_within(o[fine], e[fine], bound[fine], "finite")
    c.table[1, 2] = -1
    o2 = ops.cached_attention(q, c.k, c.v, c.table, c.cached)
    assert torch.equal(o2[0], o[0]) and bool(o2[1].isnan().all())


@pytest.mark.parametrize("decay", [0.0, 0.75])
@pytest.mark.parametrize("dtype,H,K,Dh,S,cached", [("bf16", 40, 2, 64, 16, [300, 31, 1000]), ("fp32", 33, 1, 128, 32, [0, 500])])
def test_received_weights_of_blocks_of_many_rows(dtype, H, K, Dh, S, cached, decay):
    c, q, fresh = build(9, dtype, H, K, Dh, S, cached, weights=True)
    if decay == 0.0:
        c.w.fill_(float("nan"))
    before = c.w.clone()
    widen(c, H // K)
    _, ps = check(c, q, cached, fresh, weights=c.w, decay=decay)
    for b, n in enumerate(cached):
        page, slot = c.where(b, n + 1)
        for h in range(K):
            rows = [ps[b, i, 0] for i in range(h * (H // K), (h + 1) * (H // K))]
            got, old = sum(p for p, _ in rows), before[page, h, slot].double()
            # as in test_received_weights
            bound = got * (2 * max(s for _, s in rows) + (len(rows) + 4) * 2.0 ** -24) + (3 * 2.0 ** -24 * old if decay else 0.0) + 1e-37
            assert_within(c.w[page, h, slot], got + (decay * old if decay else 0.0), bound, "weights")


def test_weights_of_padded_rows():
    c, q, _ = build(21, "bf16", 4, 2, 64, 16, [0, 20, 40], fresh=[0, 0, 1], weights=True)
    before = c.w.clone()
    o = ops.cached_attention(q, c.k, c.v, c.table, c.cached, torch.tensor([0, 0, 1], dtype=torch.int32, device=DEV),
                             weights=c.w)
    assert not bool(o[:2].any()) and bool(o[2].any())
    for b in (0, 1):
        page, slot = c.where(b, 20)
        assert torch.equal(c.w[page, :, slot], before[page, :, slot])


@pytest.mark.parametrize("S", [16, 24])
@pytest.mark.parametrize("weights", [False, True])
def test_bad_tables(S, weights):
    """A page outside the cache, negative counts and counts beyond the table: NaN in that sequence, the others as ever."""
    cached = [100, 100, 100, 100, 100, 100]
    c, q, fresh = build(13, "bf16", 4, 2, 64, S, cached, weights=weights)
    good = ops.cached_attention(q, c.k, c.v, c.table, c.cached)
    c.table[1, 0] = c.k.size(0)
    c.table[2, 3] = -1
    c.cached[3] = -1
    c.cached[4] = 10 ** 9
    c.table[5, 100 // S + 1:] = -7     # behind the last token: not looked at
    before = c.w.clone() if weights else None
    o = ops.cached_attention(q, c.k, c.v, c.table, c.cached, weights=c.w)
    assert torch.equal(o[[0, 5]], good[[0, 5]])
    assert bool(o[1:5].isnan().all())
    if weights:  # nothing is written for counts that cannot be
        for b in (3, 4):
            page, slot = c.where(b, 100)
            assert torch.equal(c.w[page, :, slot], before[page, :, slot])


def test_query_layouts_and_number_types():
    cached = [33, 90]
    c, q, fresh = build(17, "bf16", 4, 2, 64, 16, cached, T=3)
    o, _ = check(c, q, cached, fresh)
    wide = torch.zeros((2, 3, 4, 70), dtype=q.dtype, device=DEV)
    wide[..., 3:67] = q.transpose(1, 2)
    assert torch.equal(ops.cached_attention(wide[..., 3:67].transpose(1, 2), c.k, c.v, c.table, c.cached), o)
    assert torch.equal(ops.cached_attention(q.transpose(2, 3).contiguous().transpose(2, 3), c.k, c.v, c.table, c.cached), o)
    assert torch.equal(ops.cached_attention(q, c.k, c.v, c.table.long(), c.cached.long()), o)
    assert torch.equal(ops.cached_attention(q, c.k, c.v, c.table.t().contiguous().t(), c.cached), o)
    same = q[:, :1].expand(-1, 4, -1, -1)
    assert torch.equal(ops.cached_attention(same, c.k, c.v, c.table, c.cached),
                       ops.cached_attention(same.contiguous(), c.k, c.v, c.table, c.cached))


def test_empty_calls():
    c, q, _ = build(19, "bf16", 4, 2, 64, 16, [5])
    assert ops.cached_attention(q[:0], c.k, c.v, c.table[:0], c.cached[:0]).shape == (0, 4, 1, 64)
    assert ops.cached_attention(q[:, :, :0], c.k, c.v, c.table, c.cached).shape == (1, 4, 0, 64)
    none = torch.zeros((1, 0), dtype=torch.int32, device=DEV)
    o = ops.cached_attention(q, c.k, c.v, none, torch.zeros_like(c.cached), torch.zeros_like(c.cached))
    assert not bool(o.any())
    assert bool(ops.cached_attention(q, c.k, c.v, none, torch.zeros_like(c.cached)).isnan().all())


def test_same_result_every_time():
    cached = [700, 3, 1500]
    c, q, _ = build(23, "bf16", 8, 2, 128, 64, cached, weights=True)
    first, w = None, c.w.clone()
    for _ in range(3):
        c.w.copy_(w)
        o = ops.cached_attention(q, c.k, c.v, c.table, c.cached, weights=c.w)
        first = (o, c.w.clone()) if first is None else first
        assert torch.equal(o, first[0]) and torch.equal(c.w, first[1])


def test_one_page_of_several_sequences():
    """A shared beginning: two sequences read the same pages."""
    c, q, fresh = build(29, "bf16", 4, 2, 64, 16, [40, 47])
    c.table[1, :2] = c.table[0, :2]
    check(c, q, [40, 47], fresh)


@pytest.mark.parametrize("weights", [False, True])
def test_graphs(weights):
    """Two captured calls of different caches, replayed in turn with counts that grow in between."""
    made = [build(s, "bf16", 8, 2, 64, 16, [3, 200], room=400, weights=weights) for s in (31, 32)]
    for c, _, _ in made:
        c.put(gen(1), [400, 400])
        if weights:
            c.w.zero_()
    graphs = []
    for c, q, _ in made:
        ops.cached_attention(q, c.k, c.v, c.table, c.cached, weights=c.w)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = ops.cached_attention(q, c.k, c.v, c.table, c.cached, weights=c.w)
        graphs.append((graph, o))
    for step in range(4):
        for (c, q, _), (graph, o) in zip(made, graphs):
            w = c.w.clone() if weights else None
            graph.replay()
            eager = ops.cached_attention(q, c.k, c.v, c.table, c.cached, weights=w)
            torch.cuda.synchronize()
            assert torch.equal(o, eager)
            assert not weights or torch.equal(c.w, w)
            c.cached += 17
            c.k[c.table[0, 0].long()] *= 0.5


def test_a_pool_without_pages():
    """Tokens have nowhere to be: NaN; a sequence without new ones has zeros."""
    c, q, _ = build(57, "bf16", 4, 2, 64, 16, [5, 5], weights=True)
    k, v, w = c.k[:0], c.v[:0], c.w[:0]
    fresh = torch.tensor([1, 0], dtype=torch.int32, device=DEV)
    for kw in ({}, dict(weights=w)):
        o = ops.cached_attention(q, k, v, c.table, c.cached, fresh=fresh, **kw)
        assert bool(o[0].isnan().all()) and not bool(o[1].any())


def test_two_streams():
    made = [build(s, "bf16", 8, 2, 64, 16, [1000, 40, 3000]) for s in (41, 42)]
    want = [ops.cached_attention(q, c.k, c.v, c.table, c.cached) for c, q, _ in made]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    got = []
    for _ in range(5):
        for s, (c, q, _) in zip(streams, made):
            with torch.cuda.stream(s):
                got.append(ops.cached_attention(q, c.k, c.v, c.table, c.cached))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 2])


def test_far_pages():
    """A page whose elements lie beyond 2^32 of the first."""
    S, Dh = 16, 64
    P = (1 << 32) // (S * Dh) + 64
    pool = torch.empty((P, 1, S, Dh), dtype=torch.bfloat16, device=DEV)
    g = gen(43)
    for far in (P - 3, P - 40):
        pool[far] = torch.randn((1, S, Dh), generator=g).to(torch.bfloat16).to(DEV)
    c = Cache(g, torch.bfloat16, 1, Dh, S, [20], 32)
    c.k = c.v = pool
    c.table = torch.tensor([[P - 3, P - 40]], dtype=torch.int32, device=DEV)
    q = queries(g, 1, 2, 1, Dh, torch.bfloat16)
    check(c, q, [20], [1])


def test_compiled_call():
    c, q, _ = build(47, "bf16", 4, 2, 64, 16, [33, 90], weights=True)
    want_w = c.w.clone()
    want = ops.cached_attention(q, c.k, c.v, c.table, c.cached, weights=want_w, decay=0.5)

    def f(q, k, v, table, cached, w):
        return ops.cached_attention(q, k, v, table, cached, weights=w, decay=0.5) * 1.0

    got = torch.compile(f, backend="aot_eager")(q, c.k, c.v, c.table, c.cached, c.w)
    assert torch.equal(got, want) and torch.equal(c.w, want_w)


def test_refusals():
    c, q, _ = build(51, "bf16", 4, 2, 64, 16, [33, 90], weights=True)
    a = (c.k, c.v, c.table, c.cached)

    def refused(word, q=q, k=c.k, v=c.v, table=c.table, cached=c.cached, **kw):
        with pytest.raises(RuntimeError, match=word):
            ops.cached_attention(q, k, v, table, cached, **kw)

    refused("must be \\[B, heads", q=q[0])
    refused("do not share", q=q[:, :3])
    refused("do not share", q=q[..., :32])
    refused("one dtype", q=q.float())
    refused("one dtype", v=c.v.half())
    refused("one shape", v=c.v[:, :, :8])
    refused("same strides", v=c.v.transpose(1, 2).contiguous().transpose(1, 2))
    refused("block_table must be", table=c.table[:1])
    refused("block_table must be integers", table=c.table.float())
    refused("cached must be", cached=c.cached[:1])
    refused("cached must be integers", cached=c.cached.float())
    refused("fresh must be", fresh=c.cached[:1])
    refused("all tensors must be on", table=c.table.cpu())
    refused("decay", weights=c.w, decay=1.5)
    refused("decay", weights=c.w, decay=float("nan"))
    refused("scale", scale=float("inf"))
    refused("scale", scale=-2e38)
    refused("weights must be", weights=c.w.half())
    refused("weights must be", weights=c.w[:, :1])
    refused("overlap", weights=c.w[:1].expand(c.w.size(0), -1, -1))
    refused("single new token", q=q.expand(-1, -1, 2, -1), weights=c.w)
    refused("not supported", q=q.double(), k=c.k.double(), v=c.v.double())
    big = torch.zeros((2, 1, 16, 257), dtype=torch.bfloat16, device=DEV)
    refused("above 256", q=big[:, :, :1], k=big, v=big)
    with pytest.raises(RuntimeError, match="no backward"):
        ops.cached_attention(q.clone().requires_grad_(True), *a)
    with torch.no_grad():
        assert torch.equal(ops.cached_attention(q.clone().requires_grad_(True), *a), ops.cached_attention(q, *a))
