"""Generation on the GPU in the modes that programs run it in: under autocast, without a synchronization, and each of its calls
against the operators' definitions."""

import pytest
import torch

import attnres_decoder as AD

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
