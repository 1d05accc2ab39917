"""Generation on the GPU in the modes that programs run it in: under autocast, without a synchronization, and each of its calls
against the operators' definitions."""

import pytest
import torch

import attnres_decoder as AD
import attnres_ops as ops

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
