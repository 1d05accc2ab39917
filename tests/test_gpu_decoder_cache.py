"""Generation on the GPU: the cache's three operators as the decoder runs them together, and the decoder against itself
without a cache."""

from types import SimpleNamespace

import pytest
import torch

import attnres_decoder as AD
import attnres_ops as ops
from attnres_cache import PagedCache
from cache_util import append_ref, assert_within, attend_ref, evict_ref
from oracle import attnres_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
CFG = dict(n_layer=3, n_head=2, n_embd=128, mlp_hidden_dim=160, vocab_size=64, block_size=256, attnres_num_blocks=2,
           lrid_rank=32, attn_res_query_init="normal", init_std=0.05)
# A hidden state is rms-normed, of size 1.  fp32: six sublayers of products of at most 160 terms, 160 u of the sums'
# magnitude each at worst, 6e-5 in all.  bf16: in each sublayer about eight roundings of half a step, 2^-8, that the two ways
# place differently: 6 * 8 / 256 at worst where all of them add up.
MOST = {torch.float32: 1e-4, torch.bfloat16: 0.19}


def model(dtype, **kw):
    torch.manual_seed(3)
    return AD.Decoder(AD.DecoderConfig(**{**CFG, **kw})).to(DEV, dtype)


def close(a, b, dtype):
    assert bool(torch.isfinite(a).all())
    assert float((a.float() - b.float()).abs().max()) <= MOST[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kw", [dict(), dict(use_attnres=False), dict(fuse_qkv_rotary=True, fuse_swiglu=True)])
@pytest.mark.parametrize("pieces", [[100], [1] * 12, [60, 1, 1, 7, 31], [1, 99]])
def test_pieces_of_a_sequence(dtype, kw, pieces):
    m = model(dtype, **kw)
    idx = torch.randint(0, 64, (3, sum(pieces)), device=DEV)
    with torch.no_grad():
        want = m(idx, return_hidden=True)
        cache, got, at = m.new_cache(3, page_size=16), [], 0
        for n in pieces:
            got.append(m(idx[:, at:at + n], return_hidden=True, cache=cache))
            at += n
    close(torch.cat(got, 1), want, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_padded_prompts_and_steps(dtype):
    m = model(dtype)
    lengths = [90, 1, 64, 33]
    idx = torch.randint(0, 64, (4, 90), device=DEV)
    more = torch.randint(0, 64, (4, 5), device=DEV)
    with torch.no_grad():
        cache = m.new_cache(4)
        got = [m(idx, return_hidden=True, cache=cache, fresh=lengths)]
        got += [m(more[:, t:t + 1], return_hidden=True, cache=cache) for t in range(5)]
        for b, n in enumerate(lengths):
            want = m(torch.cat([idx[b, :n], more[b]])[None], return_hidden=True)[0]
            close(torch.cat([got[0][b, :n], *(g[b] for g in got[1:])]), want, dtype)


def test_generate_with_and_without_a_budget():
    m = model(torch.bfloat16)
    idx = torch.randint(0, 64, (3, 40), device=DEV)
    plain = m.generate(idx, 30, lengths=[40, 7, 20])
    # a budget that is never reached changes nothing: the weights are only added up beside
    assert torch.equal(m.generate(idx, 30, lengths=[40, 7, 20], budget=200), plain)
    cache = m.new_cache(3, page_size=8, weights=True, spare_tokens=32)
    out = m.generate(idx, 100, lengths=[40, 7, 20], cache=cache, budget=32, recent=8)
    assert out.shape == (3, 100) and max(cache.lengths) < 40 and cache.next_positions == [139, 106, 119]
    assert cache.cached.tolist() == cache.lengths and cache.positions.tolist() == cache.next_positions
    assert torch.equal(out[:, 0], plain[:, 0])


def test_generate_in_inference_mode():
    m = model(torch.bfloat16)
    idx = torch.randint(0, 64, (2, 30), device=DEV)
    kw = dict(budget=24, recent=4)
    plain = m.generate(idx, 40, cache=m.new_cache(2, page_size=8, weights=True, spare_tokens=24), **kw)
    with torch.inference_mode():
        inside = m.generate(idx, 40, cache=m.new_cache(2, page_size=8, weights=True, spare_tokens=24), **kw)
    assert torch.equal(inside, plain)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_the_operators_together(dtype):
    """Prompts, steps that count what tokens receive, evictions, more steps: each call against its definition on the
    cache as the calls before it left it."""
    H, K, Dh, S, B = 6, 2, 64, 16, 3
    g = torch.Generator().manual_seed(11)
    c = PagedCache(1, K, Dh, B, 160, page_size=S, dtype=dtype, device=DEV, weights=True, spare_tokens=48)
    inv = 10000.0 ** (-torch.arange(0, Dh, 2, dtype=torch.float64) / Dh)
    angle = torch.outer(torch.arange(400, dtype=torch.float64), inv)
    sin, cos = angle.sin().float().to(DEV), angle.cos().float().to(DEV)
    k, v, w = c.k[0], c.v[0], c.weights[0]

    def get(t, b, n):
        j = torch.arange(n, device=DEV)
        return t[c.table[b].long()[j // S], :, j % S].transpose(0, 1)

    view = SimpleNamespace(S=S, K=K, k=k, v=v, get=get)  # as the reference forms read it

    def call(T, fresh=None):
        new = [T] * B if fresh is None else fresh
        c.reserve(new)
        qkv = torch.randn((B, T, (H + 2 * K) * Dh), generator=g).to(dtype).to(DEV)
        f = None if fresh is None else torch.tensor(fresh, dtype=torch.int32, device=DEV)
        q = ops.qkv_norm_rotary_cached(qkv, H, sin, cos, k, v, c.table, c.cached, fresh=f, positions=c.positions, weights=w)
        at = torch.tensor(c.next_positions, device=DEV)[:, None] + torch.arange(T, device=DEV)
        e, bound = append_ref(qkv, H, K, sin, cos, at)
        old = w.clone()
        o = ops.cached_attention(q, k, v, c.table, c.cached, fresh=f, weights=w if T == 1 else None, decay=0.9)
        ref, most, ps = attend_ref(view, q, c.lengths, new, Dh ** -0.5)
        assert_within(o, ref, most, "attention")
        for b, n in enumerate(new):
            assert_within(q[b, :, :n], e[b, :n, :H].transpose(0, 1), bound[b, :n, :H].transpose(0, 1), "queries")
            assert_within(get(k, b, c.lengths[b] + n)[:, c.lengths[b]:], e[b, :n, H:].transpose(0, 1),
                          bound[b, :n, H:].transpose(0, 1), "keys")
            if T == 1 and n:
                for h in range(K):
                    rows = [ps[b, i, 0] for i in range(h * (H // K), (h + 1) * (H // K))]
                    was = get(old[..., None], b, c.lengths[b] + 1)[h, :, 0].double()
                    want = sum(p for p, _ in rows) + 0.9 * was
                    have = get(w[..., None], b, c.lengths[b] + 1)[h, :, 0]
                    share = 2 * max(s for _, s in rows) + 8 * 2.0 ** -24
                    # (0.9 in fp32 is off by half a step of it too)
                    assert_within(have, want, share * want + 1e-30, "weights")
        c.advance(new)

    call(70, fresh=[70, 0, 33])
    call(9, fresh=[0, 9, 4])
    for _ in range(4):
        call(1)
    for budget, recent in ((48, 16), (30, 0)):
        before, old_table, lengths = w.clone(), c.table.clone(), list(c.lengths)
        moved = k.clone()
        (kept,) = c.evict(ops, budget, recent)
        for b, n in enumerate(lengths):
            for h in range(K):
                j = torch.arange(n, device=DEV)
                weights = before[old_table[b].long()[j // S], h, j % S].tolist()
                want = evict_ref(weights, n, budget, recent)
                assert kept[b, h, :len(want)].tolist() == want and bool((kept[b, h, len(want):] == -1).all())
                src = torch.tensor(want, device=DEV)
                assert torch.equal(get(k, b, len(want))[h], moved[old_table[b].long()[src // S], h, src % S])
        assert c.lengths == [min(n, budget) for n in lengths] == c.cached.tolist()
        for _ in range(3):
            call(1)
        call(3)


def test_captured_steps():
    """A step captured once and replayed, against eager steps of a cache of the same pages."""
    m = model(torch.bfloat16)
    idx = torch.randint(0, 64, (2, 30), device=DEV)
    tokens = torch.randint(0, 64, (12, 2, 1), device=DEV)
    caches = [m.new_cache(2, page_size=16, weights=True) for _ in range(2)]
    with torch.no_grad():
        for c in caches:
            m(idx, cache=c)
            c.reserve(20)
            m(tokens[0], cache=c)
        eager, held = caches
        token = tokens[1].clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = m(token, cache=held)
        # (the capture advanced the host's counts once, and the device's not at all: its first replay does)
        for i in range(1, 12):
            token.copy_(tokens[i])
            graph.replay()
            if i > 1:
                held.replayed(1)
            want = m(tokens[i], cache=eager)
            torch.cuda.synchronize()
            assert torch.equal(logits, want)
            assert held.cached.tolist() == held.lengths == eager.lengths
            for a, b in ((held.k, eager.k), (held.v, eager.v), (held.weights, eager.weights)):
                assert torch.equal(held.table, eager.table)
                used = torch.arange(16 * held.table.size(1), device=DEV)[:held.lengths[0]]
                for s in range(2):
                    p = held.table[s].long()[used // 16]
                    assert torch.equal(a[:, p, :, used % 16], b[:, p, :, used % 16])


def test_a_cache_needs_no_gradients():
    m = model(torch.bfloat16)
    with pytest.raises(RuntimeError, match="no backward"):
        m(torch.randint(0, 64, (2, 3), device=DEV), cache=m.new_cache(2))


def test_oracle_forms_agree():
    """The oracle's cached attention, which stands in for the kernels on the CPU, against the kernel."""
    g = torch.Generator().manual_seed(2)
    c = PagedCache(1, 2, 32, 2, 60, page_size=8, dtype=torch.float32, device="cpu")
    for t in (c.k, c.v):
        t.copy_(torch.randn(t.shape, generator=g))
    c.reserve([50, 20])
    q = torch.randn((2, 4, 2, 32), generator=g)
    cached = torch.tensor([48, 18], dtype=torch.int32)
    want = O.cached_attention_ref(q, c.k[0], c.v[0], c.table, cached)
    got = ops.cached_attention(q.to(DEV), c.k[0].to(DEV), c.v[0].to(DEV), c.table.to(DEV), cached.to(DEV))
    # fp32 both: sums of 32 products and of 50 weighted values in different orders
    assert float((got.cpu() - want).abs().max()) <= 64 * 2.0 ** -24 * 8 * float(c.v.abs().max())
