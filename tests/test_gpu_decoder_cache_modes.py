"""Generation on the GPU in the modes that programs run it in: under autocast, without a synchronization, and each of its calls
against the operators' definitions."""

from types import SimpleNamespace

import pytest
import torch

import attnres_decoder as AD
import attnres_ops as ops
from attnres_cache import send
from cache_util import append_ref, assert_within, attend_ref, evict_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
CFG = dict(n_layer=3, n_head=2, n_embd=128, mlp_hidden_dim=160, vocab_size=64, block_size=256, attnres_num_blocks=2,
           lrid_rank=32, attn_res_query_init="normal", init_std=0.05)


def model(dtype, ops=None, **kw):
    torch.manual_seed(3)
    return AD.Decoder(AD.DecoderConfig(**{**CFG, **kw}), ops=ops).to(DEV, dtype)


def test_fp32_parameters_under_autocast():
    """The cached decoder rounds where the other one does or at fewer places, so against the model in fp32 its mean square error is
    at most the other's but for chance; 1.5 as for the fused sublayers."""
    m = model(F32, use_attnres=False)
    idx = torch.randint(0, 64, (3, 60), device=DEV)
    with torch.no_grad():
        exact = m(idx, return_hidden=True)
        with torch.autocast(DEV, BF):
            eager = m(idx, return_hidden=True)
            cache, got, at = m.new_cache(3, page_size=16), [], 0
            assert cache.k.dtype == cache.v.dtype == BF
            for n in (30, 1, 1, 20, 8):
                got.append(m(idx[:, at:at + n], return_hidden=True, cache=cache))
                at += n
        wide = m.new_cache(3, page_size=16)
        assert wide.k.dtype == F32
        plain = torch.cat([m(idx[:, :30], return_hidden=True, cache=wide), m(idx[:, 30:], return_hidden=True, cache=wide)], 1)
    errors = [float((h.float() - exact).norm()) for h in (torch.cat(got, 1), eager)]
    assert 0.0 < errors[0] <= 1.5 * errors[1], errors
    assert float((plain - exact).abs().max()) <= 1e-4  # (fp32 as it was)


@pytest.mark.parametrize("kw", [dict(budget=12, recent=4), dict()])
def test_generate_under_autocast(kw):
    m = model(F32, use_attnres=False)
    idx = torch.randint(0, 64, (2, 9), device=DEV)
    with torch.autocast(DEV, BF):
        out = m.generate(idx, 60, lengths=[9, 4], **kw)
        # a cache of another dtype than the projection's: its own is the dtype of heads and attention
        own = m.generate(idx, 5, cache=m.new_cache(2, dtype=F32))
    assert out.shape == (2, 60) and own.shape == (2, 5)
    assert m.generate(idx, 5, cache=m.new_cache(2, dtype=BF)).shape == (2, 5)


def test_steps_without_a_synchronization():
    """Steps that take pages, steps of some sequences alone, evictions: nothing waits for the GPU."""
    m = model(BF)
    idx = torch.randint(0, 64, (3, 20), device=DEV)
    lengths = [20, 3, 11]
    cache = m.new_cache(3, page_size=4, weights=True, spare_tokens=40)

    def work():
        m(idx, cache=cache, fresh=lengths)
        for _ in range(9):
            m(idx[:, :1], cache=cache)
        m(idx[:, :5], cache=cache, fresh=[5, 0, 2])
        cache.evict(ops, 16, 4)
        m(idx[:, :1], cache=cache)
        m.generate(idx, 12, cache=cache, lengths=lengths, budget=24, recent=3)
        for b in range(3):
            cache.drop(b)

    with torch.no_grad():
        work()
        torch.cuda.synchronize()
        torch.cuda.set_sync_debug_mode("error")
        try:
            work()
        finally:
            torch.cuda.set_sync_debug_mode("default")


def test_a_captured_step_takes_no_pages_and_no_counts(monkeypatch):
    """A replay would copy from host memory that has long been used again: refused, with nothing taken."""
    m = model(BF)
    idx = torch.randint(0, 64, (2, 6), device=DEV)
    cache = m.new_cache(2, page_size=4, weights=True, spare_tokens=8)
    with torch.no_grad():
        m(idx, cache=cache)
        before = list(cache._free), [list(o) for o in cache._owned], list(cache.lengths), cache.table.clone()
        with monkeypatch.context() as patch:
            patch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
            for call in (lambda: m(idx[:, :3], cache=cache),                       # a page more
                         lambda: m(idx[:, :2], cache=cache, fresh=[2, 1]),         # counts
                         lambda: cache.advance([1, 0]), lambda: cache.evict(ops, 4, 1), lambda: cache.drop(0)):
                with pytest.raises(RuntimeError, match="captured"):
                    call()
        assert before[:3] == (cache._free, cache._owned, cache.lengths) and torch.equal(cache.table, before[3])
        want = m(torch.cat([idx, idx[:, :3]], 1))[:, 6:]
        got = m(idx[:, :3], cache=cache)
    # (bf16 hidden states, as far apart as the ways of computing them are)
    assert got.shape == want.shape and bool(torch.isfinite(got).all())


def test_numbers_sent_while_the_stream_is_busy():
    """Each from memory of its own until it has arrived, however far ahead the host is."""
    like = torch.zeros((1,), dtype=torch.int32, device=DEV)
    x = torch.randn((4096, 4096), device=DEV)
    for _ in range(2):  # (the second time from memory that the first one used)
        y = x
        for _ in range(20):
            y = (x @ y) * 1e-2
        sent = [send([i, i * 7 + 1, -i], like) for i in range(500)]
        assert torch.equal(torch.stack(sent).cpu(), torch.tensor([[i, i * 7 + 1, -i] for i in range(500)], dtype=torch.int32))


class Checked:
    """The drop-in module's functions; the cache's three are held against their definitions on what they were given."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return getattr(ops, name)

    @staticmethod
    def _view(k, v, table):
        S = k.size(2)

        def get(t, b, n):
            j = torch.arange(n, device=DEV)
            return t[table[b].long()[j // S], :, j % S].transpose(0, 1)

        return SimpleNamespace(S=S, K=k.size(1), k=k, v=v, get=get)

    def qkv_norm_rotary_cached(self, qkv, H, sin, cos, k, v, table, cached, fresh=None, positions=None, qk_norm=True, weights=None,
                               return_heads=False):
        out = ops.qkv_norm_rotary_cached(qkv, H, sin, cos, k, v, table, cached, fresh=fresh, positions=positions, qk_norm=qk_norm,
                                         weights=weights, return_heads=return_heads)
        (B, T, _), K, c = qkv.shape, k.size(1), self._view(k, v, table)
        half = sin.size(-1)
        at = (positions[:, None] + torch.arange(T, device=DEV)).long()
        e, bound = append_ref(qkv, H, K, sin.view(-1, half), cos.view(-1, half), at.clamp(max=sin.numel() // half - 1), qk_norm=qk_norm)
        q = out[0] if return_heads else out
        values = qkv.view(B, T, H + 2 * K, 2 * half)[:, :, H + K:]
        for b in range(B):
            n, f = int(cached[b]), T if fresh is None else int(fresh[b])
            assert_within(q[b, :, :f], e[b, :f, :H].transpose(0, 1), bound[b, :f, :H].transpose(0, 1), "queries")
            assert_within(c.get(k, b, n + f)[:, n:], e[b, :f, H:].transpose(0, 1), bound[b, :f, H:].transpose(0, 1), "keys")
            assert torch.equal(c.get(v, b, n + f)[:, n:], values[b, :f].transpose(0, 1))
        self.calls.append("append")
        return out

    def cached_attention(self, q, k, v, table, cached, fresh=None, weights=None):
        (B, H, T, Dh), c = q.shape, self._view(k, v, table)
        old = None if weights is None else weights.clone()
        o = ops.cached_attention(q, k, v, table, cached, fresh=fresh, weights=weights)
        new = [T] * B if fresh is None else fresh.tolist()
        e, bound, ps = attend_ref(c, q, cached.tolist(), new, Dh ** -0.5)
        assert_within(o, e, bound, "attention")
        if weights is not None:
            for b, n in enumerate(cached.tolist()):
                for h in range(c.K if new[b] else 0):
                    rows = [ps[b, i, 0] for i in range(h * (H // c.K), (h + 1) * (H // c.K))]
                    was = c.get(old[..., None], b, n + 1)[h, :, 0].double()
                    share = 2 * max(s for _, s in rows) + 8 * 2.0 ** -24
                    want = sum(p for p, _ in rows) + was
                    assert_within(c.get(weights[..., None], b, n + 1)[h, :, 0], want, share * want + 1e-30, "weights")
        self.calls.append("attend")
        return o

    def evict_cached_tokens(self, k, v, weights, table, cached, new, budget, recent):
        S, old = k.size(2), [t.clone() for t in (k, v, weights)]
        kept, left = ops.evict_cached_tokens(k, v, weights, table, cached, new, budget, recent)
        lengths = cached.tolist()
        assert left.tolist() == [min(n, budget) for n in lengths]
        for b, n in enumerate(lengths):
            j = torch.arange(n, device=DEV)
            page, slot = table[b].long()[j // S], j % S
            for h in range(k.size(1)):
                e = evict_ref(old[2][page, h, slot].tolist(), n, budget, recent)
                assert kept[b, h].tolist() == e + [-1] * (budget - len(e))
                i = torch.arange(len(e), device=DEV)
                for t, was in zip((k, v, weights), old):
                    assert torch.equal(t[new[b].long()[i // S], h, i % S], was[page[e], h, slot[e]])
        self.calls.append("evict")
        return kept, left


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("kw", [dict(), dict(use_attnres=False)])
def test_every_call_of_a_generation_within_a_budget(dtype, kw):
    checked = Checked()
    m = model(dtype, ops=checked, **kw)
    idx = torch.randint(0, 64, (3, 30), device=DEV)
    cache = m.new_cache(3, page_size=8, weights=True, spare_tokens=24)
    out = m.generate(idx, 24, lengths=[30, 6, 17], cache=cache, budget=24, recent=6)
    # a second turn of several tokens over what is left, and more of them
    more = m.generate(idx[:, :7], 9, lengths=[7, 2, 5], cache=cache, budget=24, recent=6)
    assert out.shape == (3, 24) and more.shape == (3, 9)
    layers = CFG["n_layer"]
    assert checked.calls.count("append") == 33 * layers and checked.calls.count("attend") == 32 * layers
    assert checked.calls.count("evict") >= 2 * layers
    assert cache.next_positions == [30 + 23 + 7 + 8, 6 + 23 + 2 + 8, 17 + 23 + 5 + 8] == cache.positions.tolist()
    assert cache.cached.tolist() == cache.lengths and max(cache.lengths) < 32
