"""qkv_norm_rotary_cached against its definition in 64 bits: what is written where, and that nothing else is."""

import pytest
import torch

import attnres_ops as ops
from cache_util import Cache, append_ref, assert_within

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ROWS = 600


def gen(seed):
    return torch.Generator().manual_seed(seed)


def tables(Dh, dtype, rows=ROWS):
    inv = 10000.0 ** (-torch.arange(0, Dh, 2, dtype=torch.float64) / Dh)
    a = torch.outer(torch.arange(rows, dtype=torch.float64), inv)
    return a.sin().to(dtype).to(DEV), a.cos().to(dtype).to(DEV)


def build(seed, dtype, H, K, Dh, S, cached, T, layout="dense", room=None, weights=False, table="fp32"):
    g = gen(seed)
    c = Cache(g, DT[dtype], K, Dh, S, cached, max(cached) + T if room is None else room, layout, fill=0.125, weights=weights)
    qkv = (torch.randn((len(cached), T, H + 2 * K, Dh), generator=g) *
           torch.exp2(torch.randn((H + 2 * K, 1), generator=g))).flatten(2).to(DT[dtype]).to(DEV)
    return c, qkv, *tables(Dh, DT[table])


def check(c, qkv, H, sin, cos, cached, fresh=None, positions=None, qk_norm=True, weights=False, heads=True):
    B, T, _ = qkv.shape
    K, Dh = c.K, c.Dh
    before = [c.k.clone(), c.v.clone(), None if c.w is None else c.w.clone()]
    kw = {} if fresh is None else dict(fresh=torch.tensor(fresh, dtype=torch.int32, device=DEV))
    if positions is not None:
        kw["positions"] = torch.tensor(positions, dtype=torch.int32, device=DEV)
    out = ops.qkv_norm_rotary_cached(qkv, H, sin, cos, c.k, c.v, c.table, c.cached, qk_norm=qk_norm,
                                     weights=c.w if weights else None, return_heads=heads, **kw)
    q, k, v = out if heads else (out, None, None)
    at = torch.tensor(cached if positions is None else positions, device=DEV)[:, None] + torch.arange(T, device=DEV)
    e, bound = append_ref(qkv, H, K, sin, cos, at, qk_norm=qk_norm)
    fresh = [T] * B if fresh is None else fresh
    for b, f in enumerate(fresh):
        e[b, f:] = 0
        bound[b, f:] = 0
    assert q.shape == (B, H, T, Dh) and q.is_contiguous()
    assert_within(q, e[:, :, :H].transpose(1, 2), bound[:, :, :H].transpose(1, 2), "q")
    values = qkv.view(B, T, H + 2 * K, Dh)[:, :, H + K:]
    if heads:
        assert_within(k, e[:, :, H:].transpose(1, 2), bound[:, :, H:].transpose(1, 2), "k")
        assert torch.equal(v, values.transpose(1, 2)) and v.data_ptr() == values.data_ptr()
    for b, f in enumerate(fresh):
        page, slot = c.where(b, cached[b] + f)
        page, slot = page[cached[b]:], slot[cached[b]:]
        assert_within(c.k[page, :, slot], e[b, :f, H:], bound[b, :f, H:], "cached keys")
        if heads:
            assert torch.equal(c.k[page, :, slot], k[b, :, :f].transpose(0, 1))
        assert torch.equal(c.v[page, :, slot], values[b, :f])
        before[0][page, :, slot] = c.k[page, :, slot]
        before[1][page, :, slot] = values[b, :f]
        if weights:
            before[2][page, :, slot] = 0
    assert torch.equal(c.k, before[0]) and torch.equal(c.v, before[1]), "nothing else is written"
    assert c.w is None or torch.equal(c.w, before[2])
    return out


@pytest.mark.parametrize("dtype,table", [("bf16", "fp32"), ("bf16", "bf16"), ("fp16", "fp32"), ("fp16", "fp16"), ("fp32", "fp32")])
@pytest.mark.parametrize("H,K,Dh,S", [
    (12, 12, 64, 64), (8, 2, 128, 16), (5, 5, 40, 24), (3, 1, 256, 7), (2, 2, 6, 5), (1, 1, 2, 1), (7, 7, 20, 33), (4, 1, 32, 100),
    (2, 1, 200, 16)])
@pytest.mark.parametrize("T", [1, 9])
def test_shapes(dtype, table, H, K, Dh, S, T):
    cached = [0, 15, 16, 101, 7]
    c, qkv, sin, cos = build(H * 37 + Dh, dtype, H, K, Dh, S, cached, T, table=table)
    check(c, qkv, H, sin, cos, cached, heads=T > 1)


@pytest.mark.parametrize("layout", ["tokens", "layer", "odd"])
@pytest.mark.parametrize("dtype,Dh", [("bf16", 64), ("fp32", 40), ("fp16", 128)])
def test_layouts(layout, dtype, Dh):
    cached = [0, 30, 63]
    c, qkv, sin, cos = build(3, dtype, 4, 2, Dh, 16, cached, 40, layout, weights=True)
    check(c, qkv, 4, sin, cos, cached, weights=True)


@pytest.mark.parametrize("weights", [False, True])
def test_padded_batch_and_positions(weights):
    cached, T = [0, 40, 9, 100], 33
    c, qkv, sin, cos = build(5, "bf16", 6, 3, 64, 16, cached, T, weights=weights)
    check(c, qkv, 6, sin, cos, cached, fresh=[T, 0, 7, 1], positions=[0, 300, 17, 560], weights=weights)


def test_without_norm():
    c, qkv, sin, cos = build(7, "fp32", 4, 4, 64, 16, [3, 3], 5)
    check(c, qkv, 4, sin, cos, [3, 3], qk_norm=False)


def test_projection_layouts_and_number_types():
    cached = [3, 20]
    c, qkv, sin, cos = build(9, "bf16", 4, 2, 64, 16, cached, 5)
    want = check(c, qkv, 4, sin, cos, cached)
    for x in (qkv.transpose(0, 1).contiguous().transpose(0, 1),
              torch.cat([qkv, qkv], -1)[..., :qkv.size(-1)],
              torch.cat([qkv[..., :1], qkv], -1)[..., 1:]):
        c.k.fill_(0.125)
        got = ops.qkv_norm_rotary_cached(x, 4, sin.view(1, 1, ROWS, 32), cos.view(1, 1, ROWS, 32), c.k, c.v, c.table.long(),
                                         c.cached.long(), return_heads=True)
        # (rows that start anywhere take single values, whose norm sums in another order)
        for a, b in zip(got, want):
            assert float((a.float() - b.float()).abs().max()) <= 2.0 ** -7 * float(b.float().abs().max())
    same = qkv[:1].expand(2, -1, -1)
    a = ops.qkv_norm_rotary_cached(same, 4, sin, cos, c.k, c.v, c.table, c.cached)
    b = ops.qkv_norm_rotary_cached(same.contiguous(), 4, sin, cos, c.k, c.v, c.table, c.cached)
    assert torch.equal(a, b)


def test_what_has_no_place_is_not_written():
    cached, T = [10, 10, 10, 10], 12
    c, qkv, sin, cos = build(11, "bf16", 4, 2, 64, 16, cached, T, room=32, weights=True)
    want = ops.qkv_norm_rotary_cached(qkv, 4, sin, cos, c.k, c.v, c.table, c.cached)
    filled = c.k.clone(), c.v.clone(), c.w.clone()
    c.k.fill_(0.125), c.v.fill_(0.125)
    c.table[0, 0] = -1
    c.table[1, 1] = c.k.size(0)
    c.cached[2] = 25          # tokens 7.. are beyond the table's two pages
    c.cached[3] = -5
    kept = c.k.clone(), c.v.clone(), c.w.clone()
    pos = torch.tensor(cached, dtype=torch.int32, device=DEV)
    got = ops.qkv_norm_rotary_cached(qkv, 4, sin, cos, c.k, c.v, c.table, c.cached, positions=pos, weights=c.w)
    assert torch.equal(got, want), "the queries come all the same"
    for b, tokens in ((0, range(6, 12)), (1, range(0, 6)), (2, range(0, 7)), (3, ())):
        for t in tokens:
            j = int(c.cached[b]) + t
            page, slot = int(c.table[b, j // 16]), j % 16
            kept[0][page, :, slot] = c.k[page, :, slot]
            kept[1][page, :, slot] = qkv.view(4, T, 8, 64)[b, t, 6:]
            kept[2][page, :, slot] = 0
            assert not bool((c.k[page, :, slot] == 0.125).all())
    assert torch.equal(c.k, kept[0]) and torch.equal(c.v, kept[1]) and torch.equal(c.w, kept[2])
    del filled


def test_rows_outside_the_tables():
    c, qkv, sin, cos = build(13, "bf16", 4, 2, 64, 16, [3, 3, 3], 2)
    pos = torch.tensor([ROWS - 1, -1, 5], dtype=torch.int32, device=DEV)
    q, k, _ = ops.qkv_norm_rotary_cached(qkv, 4, sin, cos, c.k, c.v, c.table, c.cached, positions=pos, return_heads=True)
    for t in (q, k):
        bad = t.isnan().all(-1)
        assert bad.any(1).tolist() == [[False, True], [True, False], [False, False]] and bool((bad == t.isnan().any(-1)).all())
    far = torch.tensor([2 ** 40, -2 ** 40, 5], device=DEV)
    q2 = ops.qkv_norm_rotary_cached(qkv, 4, sin, cos, c.k, c.v, c.table, c.cached, positions=far)
    assert bool(q2[:2, :, :1].isnan().all()) and torch.equal(q2[2], q[2])


def test_agrees_with_the_uncached_operator():
    c, qkv, sin, cos = build(15, "bf16", 12, 12, 64, 64, [0, 0], 50)
    q, k, v = ops.qkv_norm_rotary_cached(qkv, 12, sin, cos, c.k, c.v, c.table, c.cached, return_heads=True)
    for a, b in zip((q, k, v), ops.qkv_norm_rotary(qkv, 12, sin, cos)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("Dh", [62, 86, 130, 198, 254])
@pytest.mark.parametrize("T", [1, 7])
def test_heads_of_pairs(dtype, Dh, T):
    """Widths of 4 n + 2, of up to two pairs a lane."""
    cached = [0, 15, 40]
    c, qkv, sin, cos = build(Dh, dtype, 4, 2, Dh, 16, cached, T, weights=True, table="fp32" if T > 1 else dtype)
    check(c, qkv, 4, sin, cos, cached, fresh=[T, T - 1, T], weights=True)


def test_far_pages():
    """Pages whose elements lie beyond 2^32 of the first."""
    S, Dh = 16, 64
    P = (1 << 32) // (S * Dh) + 64
    c, qkv, sin, cos = build(61, "bf16", 2, 1, Dh, S, [20], 9)
    k, v = (torch.empty((P, 1, S, Dh), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    far = torch.tensor([[P - 3, P - 40]], dtype=torch.int32, device=DEV)
    q = ops.qkv_norm_rotary_cached(qkv, 2, sin, cos, c.k, c.v, c.table, c.cached)
    assert torch.equal(ops.qkv_norm_rotary_cached(qkv, 2, sin, cos, k, v, far, c.cached), q)
    for a, b in ((k, c.k), (v, c.v)):
        assert torch.equal(a[P - 40, :, 4:13], b[int(c.table[0, 1]), :, 4:13])


def test_a_pool_without_pages():
    c, qkv, sin, cos = build(63, "bf16", 2, 1, 64, 16, [20, 3], 4)
    q = ops.qkv_norm_rotary_cached(qkv, 2, sin, cos, c.k, c.v, c.table, c.cached)
    assert torch.equal(ops.qkv_norm_rotary_cached(qkv, 2, sin, cos, c.k[:0], c.v[:0], c.table, c.cached), q)


def test_two_streams():
    """Two caches at once, each on a stream of its own."""
    made = [build(s, "bf16", 4, 2, 64, 16, [0, 100, 30], 50) for s in (65, 66)]
    want = []
    for c, qkv, sin, cos in made:
        want.append((ops.qkv_norm_rotary_cached(qkv, 4, sin, cos, c.k, c.v, c.table, c.cached), c.k.clone(), c.v.clone()))
        c.k.fill_(0.125)
        c.v.fill_(0.125)
    torch.cuda.synchronize()
    got = []
    for s, (c, qkv, sin, cos) in zip([torch.cuda.Stream(), torch.cuda.Stream()], made):
        with torch.cuda.stream(s):
            got.append(ops.qkv_norm_rotary_cached(qkv, 4, sin, cos, c.k, c.v, c.table, c.cached))
    torch.cuda.synchronize()
    for q, (c, *_), (e, k, v) in zip(got, made, want):
        assert torch.equal(q, e) and torch.equal(c.k, k) and torch.equal(c.v, v)


def test_empty_calls():
    c, qkv, sin, cos = build(17, "bf16", 4, 2, 64, 16, [3, 3], 2)
    kept = c.k.clone()
    q = ops.qkv_norm_rotary_cached(qkv[:, :0], 4, sin, cos, c.k, c.v, c.table, c.cached)
    assert q.shape == (2, 4, 0, 64)
    assert ops.qkv_norm_rotary_cached(qkv[:0], 4, sin, cos, c.k, c.v, c.table[:0], c.cached[:0]).shape == (0, 4, 2, 64)
    none = torch.zeros((2, 0), dtype=torch.int32, device=DEV)
    assert ops.qkv_norm_rotary_cached(qkv, 4, sin, cos, c.k, c.v, none, c.cached).shape == (2, 4, 2, 64)
    assert torch.equal(c.k, kept)


def test_graph():
    c, qkv, sin, cos = build(19, "bf16", 4, 2, 64, 16, [3, 30], 1, room=200)
    ops.qkv_norm_rotary_cached(qkv, 4, sin, cos, c.k, c.v, c.table, c.cached)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = ops.qkv_norm_rotary_cached(qkv, 4, sin, cos, c.k, c.v, c.table, c.cached)
    for _ in range(4):
        c.cached += 11
        k, v = c.k.clone(), c.v.clone()
        want = ops.qkv_norm_rotary_cached(qkv, 4, sin, cos, k, v, c.table, c.cached)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q, want) and torch.equal(c.k, k) and torch.equal(c.v, v)
        qkv.mul_(-0.5)


def test_compiled_call():
    c, qkv, sin, cos = build(21, "bf16", 4, 2, 64, 16, [3, 30], 2, weights=True)
    k, v, w = c.k.clone(), c.v.clone(), c.w.clone()
    want = ops.qkv_norm_rotary_cached(qkv, 4, sin, cos, k, v, c.table, c.cached, weights=w, return_heads=True)

    def f(qkv, sin, cos, k, v, table, cached, w):
        q, kk, vv = ops.qkv_norm_rotary_cached(qkv, 4, sin, cos, k, v, table, cached, weights=w, return_heads=True)
        return q * 1.0, kk, vv

    got = torch.compile(f, backend="aot_eager")(qkv, sin, cos, c.k, c.v, c.table, c.cached, c.w)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert torch.equal(c.k, k) and torch.equal(c.v, v) and torch.equal(c.w, w)


def test_refusals():
    c, qkv, sin, cos = build(23, "bf16", 4, 2, 64, 16, [3, 30], 2, weights=True)

    def refused(word, qkv=qkv, H=4, sin=sin, cos=cos, k=c.k, v=c.v, table=c.table, cached=c.cached, **kw):
        with pytest.raises(RuntimeError, match=word):
            ops.qkv_norm_rotary_cached(qkv, H, sin, cos, k, v, table, cached, **kw)

    refused("must be \\[B, T", qkv=qkv[0])
    refused("columns", H=5)
    refused("columns", H=0)
    refused("one dtype", qkv=qkv.float())
    refused("sin must be", sin=sin[:, :16])
    refused("differ in shape", sin=sin[:5])
    refused("floating-point", sin=sin.long(), cos=cos.long())
    refused("positions must be", positions=torch.zeros((2, 2), dtype=torch.int32, device=DEV))
    refused("positions must be integers", positions=torch.zeros((2,), device=DEV))
    refused("block_table must be", table=c.table[:1])
    refused("same strides", v=c.v.transpose(1, 2).contiguous().transpose(1, 2))
    refused("overlap", k=c.k[:1].expand_as(c.k), v=c.v[:1].expand_as(c.v))
    refused("all tensors must be on", cached=c.cached.cpu())
    refused("no backward", qkv=qkv.clone().requires_grad_(True))
    refused("no backward", sin=sin.clone().requires_grad_(True))
    wide = torch.zeros((2, 2, 8 * 258), dtype=torch.bfloat16, device=DEV)
    pool = torch.zeros((8, 2, 16, 258), dtype=torch.bfloat16, device=DEV)
    refused("above 256", qkv=wide, k=pool, v=pool)
    odd = torch.zeros((8, 2, 16, 63), dtype=torch.bfloat16, device=DEV)
    refused("even width", qkv=qkv[..., :8 * 63], k=odd, v=odd)
