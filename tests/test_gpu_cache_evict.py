"""evict_cached_tokens against its definition: which tokens are kept (exactly), where they go, and that nothing else changes."""

import pytest
import torch

import attnres_ops as ops
from cache_util import Cache, evict_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
INF, NAN = float("inf"), float("nan")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def build(seed, dtype, K, Dh, S, cached, budget, layout="dense", ties=True, room=None):
    g = gen(seed)
    B, per = len(cached), -(-budget // S)
    c = Cache(g, DT[dtype], K, Dh, S, cached, max(max(cached), 1) if room is None else room, layout, extra=B * per + 2,
              fill=0.125, weights=True)
    c.put(g, cached)
    if ties:
        c.w.copy_((torch.randint(0, 40, c.w.shape, generator=g) / 8.0).to(DEV))
    used = set(c.table.flatten().tolist())
    free = [p for p in range(c.k.size(0)) if p not in used]
    new = torch.tensor(free[:B * per], dtype=torch.int32).view(B, per).to(DEV)
    return c, new


def run_and_check(c, new, cached, budget, recent, table=None, cached_as=None, new_as=None):
    before = [t.clone() for t in (c.k, c.v, c.w)]
    kept, left = ops.evict_cached_tokens(c.k, c.v, c.w, c.table if table is None else table,
                                         c.cached if cached_as is None else cached_as, new if new_as is None else new_as,
                                         budget, recent)
    assert kept.dtype == left.dtype == torch.int32 and kept.shape == (c.B, c.K, budget)
    assert left.tolist() == [min(n, budget) for n in cached]
    want = [t.clone() for t in before]
    for b, n in enumerate(cached):
        page, slot = c.where(b, n)
        for h in range(c.K):
            e = evict_ref(before[2][page, h, slot].tolist(), n, budget, recent)
            assert kept[b, h].tolist() == e + [-1] * (budget - len(e)), (b, h)
            i = torch.arange(len(e), device=DEV)
            for t, old in zip(want, before):
                t[new[b].long()[i // c.S], h, i % c.S] = old[page[e], h, slot[e]]
    for name, t, e in zip("kvw", (c.k, c.v, c.w), want):
        assert torch.equal(t.nan_to_num(77.0), e.nan_to_num(77.0)), name
    return kept, left


@pytest.mark.parametrize("dtype,K,Dh,S", [("bf16", 2, 64, 16), ("fp16", 3, 40, 24), ("fp32", 1, 128, 64), ("bf16", 2, 17, 7),
                                          ("fp32", 2, 5, 1), ("bf16", 1, 256, 128), ("bf16", 2, 62, 16), ("fp16", 1, 36, 32), ("fp32", 2, 6, 16)])
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (50, 0), (50, 13), (64, 64), (130, 32)])
def test_choice_and_copies(dtype, K, Dh, S, budget, recent):
    cached = [0, 1, budget, budget + 1, 2 * budget + 5, 333]
    c, new = build(K * 7 + Dh + budget, dtype, K, Dh, S, cached, budget)
    run_and_check(c, new, cached, budget, recent)


@pytest.mark.parametrize("layout", ["tokens", "layer", "odd"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_layouts(layout, dtype):
    cached = [100, 40, 300]
    c, new = build(3, dtype, 2, 64, 16, cached, 70, layout)
    run_and_check(c, new, cached, 70, 10)


@pytest.mark.parametrize("cached,budget,recent", [([5000, 3000], 1024, 100), ([20000], 4000, 0), ([70000], 100, 50), ([9000, 16384, 12000], 2500, 300), ([16000, 5], 300, 300), ([20000, 17000], 64, 64),
                                                  ([1024, 1025, 2048, 2049], 1024, 1023)])
def test_long(cached, budget, recent):
    c, new = build(5, "bf16", 2, 8, 64, cached, budget, ties=len(cached) > 1)
    run_and_check(c, new, cached, budget, recent)


@pytest.mark.parametrize("room", [2048, 2064, 8192, 8208, 16384, 16400])
def test_tables_up_to_and_above_what_a_workgroup_holds(room):
    cached = [room, room - 1, 900]
    c, new = build(room, "bf16", 1, 8, 16, cached, 700, ties=False, room=room)
    run_and_check(c, new, cached, 700, 90)


def test_far_pages():
    """Rows from and to pages whose elements lie beyond 2^32 of the first."""
    S, Dh = 16, 64
    P = (1 << 32) // (S * Dh) + 64
    c, new = build(23, "bf16", 1, Dh, S, [40], 20)
    k, v = (torch.empty((P, 1, S, Dh), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    w = torch.zeros((P, 1, S), device=DEV)
    far = torch.tensor([[P - 3, P - 40, P - 7]], dtype=torch.int32, device=DEV)
    to = torch.tensor([[P - 50, P - 1]], dtype=torch.int32, device=DEV)
    for a, b in ((k, c.k), (v, c.v), (w, c.w)):
        a[far[0].long()] = b[c.table[0].long()]
    want = ops.evict_cached_tokens(c.k, c.v, c.w, c.table, c.cached, new, 20, 4)
    got = ops.evict_cached_tokens(k, v, w, far, c.cached, to, 20, 4)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for a, b in ((k, c.k), (v, c.v), (w, c.w)):
        assert torch.equal(a[P - 50], b[int(new[0, 0])]) and torch.equal(a[P - 1, :, :4], b[int(new[0, 1]), :, :4])


def test_a_pool_without_pages():
    """Nothing to copy; the choice is by place alone."""
    c, new = build(25, "bf16", 2, 64, 16, [40, 10], 20)
    kept, left = ops.evict_cached_tokens(c.k[:0], c.v[:0], c.w[:0], c.table, c.cached, new, 20, 5)
    assert left.tolist() == [20, 10]
    assert kept[0, 1].tolist() == list(range(15)) + list(range(35, 40)) and kept[1, 0].tolist() == list(range(10)) + [-1] * 10


def test_two_streams():
    """Two caches at once, each on a stream of its own; of tables of one workgroup a head and of several."""
    made = [build(s, "bf16", 2, 64, 16, [20000 if s == 27 else 3000, 700], 600) for s in (27, 28)]
    before = [[t.clone() for t in (c.k, c.v, c.w)] for c, _ in made]
    want = [ops.evict_cached_tokens(*t, c.table, c.cached, new, 600, 50) for t, (c, new) in zip(before, made)]
    torch.cuda.synchronize()
    got = []
    for s, (c, new) in zip([torch.cuda.Stream(), torch.cuda.Stream()], made):
        with torch.cuda.stream(s):
            got.append(ops.evict_cached_tokens(c.k, c.v, c.w, c.table, c.cached, new, 600, 50))
    torch.cuda.synchronize()
    for a, b, t, (c, _) in zip(got, want, before, made):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        assert torch.equal(c.k, t[0]) and torch.equal(c.v, t[1]) and torch.equal(c.w, t[2])


@pytest.mark.parametrize("values", [[0.0], [-0.0, 0.0], [NAN], [NAN, -INF, -1.0, 0.0], [INF, NAN, 3.0], [-INF],
                                    [1e-45, 0.0, -1e-45], [3.4e38, INF, -3.4e38], [1.0, 1.0000001]])
def test_weights_of_all_kinds(values):
    """Equal ones by their place, zeros of both signs equal, NaN below everything, subnormal ones as they are."""
    cached = [200, 90]
    c, new = build(7, "bf16", 2, 8, 16, cached, 60)
    pick = torch.randint(0, len(values), c.w.shape, generator=gen(8))
    c.w.copy_(torch.tensor(values)[pick].to(DEV))
    run_and_check(c, new, cached, 60, 20)


def test_sequences_within_the_budget_keep_their_pages():
    cached = [30, 100, 64]
    c, new = build(9, "bf16", 2, 64, 16, cached, 64, room=128)
    new[0], new[2] = c.table[0, :4], c.table[2, :4]
    run_and_check(c, new, cached, 64, 8)


def test_pages_behind_the_budget_are_not_looked_at():
    cached = [100, 90]
    c, new = build(11, "bf16", 2, 64, 16, cached, 50)
    wide = torch.full((2, 9), -3, dtype=torch.int32, device=DEV)
    wide[:, :4] = new
    table = torch.full((2, 20), 10 ** 6, dtype=torch.int32, device=DEV)
    table[:, :7] = c.table
    run_and_check(c, new, cached, 50, 5, table=table, new_as=wide[:, :5])


def test_bad_tables():
    cached = [100, 100, 100, 100]
    c, new = build(13, "bf16", 2, 64, 16, cached, 50)
    c.table[0, 0] = -1            # tokens 0..15 have no page: lowest weight, and not copied
    c.table[0, 6] = 10 ** 9       # the last four, which `recent` keeps
    new[1, 1] = c.k.size(0)       # places 16..31 have none
    c.cached[2] = -1
    c.cached[3] = 10 ** 9
    before = c.k.clone()
    kept, left = ops.evict_cached_tokens(c.k, c.v, c.w, c.table, c.cached, new, 50, 8)
    assert left.tolist() == [50, 50, 0, 0] and bool((kept[2:] == -1).all())
    for b in (0, 1):
        for h in range(2):
            places = kept[b, h].tolist()
            assert places == sorted(places) and places[-8:] == list(range(92, 100))
            assert b == 1 or min(places) >= 16
            for i, j in enumerate(places):
                to, at = int(new[b, i // 16]), i % 16
                if b == 1 and 16 <= i < 32:
                    continue
                page = int(c.table[b, j // 16])
                want = before[page, h, j % 16] if 0 <= page < c.k.size(0) else before[to, h, at]
                assert torch.equal(c.k[to, h, at], want)
    changed = (c.k != before).any(-1).any(-1).any(-1).nonzero().flatten().tolist()
    assert set(changed) <= set(new[0].tolist() + new[1].tolist())


def test_number_types_and_empty_calls():
    cached = [100, 40]
    c, new = build(15, "bf16", 2, 64, 16, cached, 50)
    run_and_check(c, new, cached, 50, 8, table=c.table.long(), cached_as=c.cached.long(), new_as=new.t().contiguous().t().long())
    kept, left = ops.evict_cached_tokens(c.k, c.v, c.w, c.table[:0], c.cached[:0], new[:0], 50, 8)
    assert kept.shape == (0, 2, 50) and left.shape == (0,)
    none = torch.zeros((2, 0), dtype=torch.int32, device=DEV)
    kept, left = ops.evict_cached_tokens(c.k, c.v, c.w, none, torch.zeros_like(c.cached), new, 50, 8)
    assert left.tolist() == [0, 0] and bool((kept == -1).all())


def test_graph():
    cached = [100, 300]
    c, new = build(17, "bf16", 2, 64, 16, cached, 64)
    ops.evict_cached_tokens(c.k, c.v, c.w, c.table, c.cached, new, 64, 8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept, left = ops.evict_cached_tokens(c.k, c.v, c.w, c.table, c.cached, new, 64, 8)
    for i in range(3):
        c.w.copy_(torch.rand(c.w.shape, generator=gen(i)).to(DEV))
        c.cached.copy_(torch.tensor([100 - 30 * i, 300 - 40 * i]))
        pools = [t.clone() for t in (c.k, c.v, c.w)]
        want = ops.evict_cached_tokens(*pools, c.table, c.cached, new, 64, 8)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept, want[0]) and torch.equal(left, want[1])
        for a, b in zip((c.k, c.v, c.w), pools):
            assert torch.equal(a, b)


def test_compiled_call():
    c, new = build(19, "bf16", 2, 64, 16, [100, 40], 50)
    pools = [t.clone() for t in (c.k, c.v, c.w)]
    want = ops.evict_cached_tokens(*pools, c.table, c.cached, new, 50, 8)
    f = torch.compile(lambda *a: [t + 0 for t in ops.evict_cached_tokens(*a, 50, 8)], backend="aot_eager")
    got = f(c.k, c.v, c.w, c.table, c.cached, new)
    for a, b in zip((*got, c.k, c.v, c.w), (*want, *pools)):
        assert torch.equal(a, b)


def test_refusals():
    c, new = build(21, "bf16", 2, 64, 16, [100, 40], 50)

    def refused(word, k=c.k, v=c.v, w=c.w, table=c.table, cached=c.cached, new=new, budget=50, recent=8):
        with pytest.raises(RuntimeError, match=word):
            ops.evict_cached_tokens(k, v, w, table, cached, new, budget, recent)

    refused("budget", budget=0)
    refused("budget", recent=51)
    refused("budget", recent=-1)
    refused("new_table", budget=65)
    refused("new_table", new=new[:1])
    refused("new_table must be integers", new=new.float())
    refused("None", w=None)
    refused("weights must be", w=c.w.half())
    refused("cached must be", cached=c.cached[:1])
    refused("all tensors must be on", new=new.cpu())
    refused("overlap", k=c.k[:1].expand_as(c.k), v=c.v[:1].expand_as(c.v))
    refused("no backward", k=c.k.clone().requires_grad_(True), v=c.v)
