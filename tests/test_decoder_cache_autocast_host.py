"""CPU checks of generation with fp32 parameters under autocast, and with a cache of a dtype of its own."""

import pytest
import torch

import attnres_decoder as AD
from test_decoder_cache_host import CFG, CacheOps

BF, F32 = torch.bfloat16, torch.float32


class Noting(CacheOps):
    def __init__(self):
        self.seen = set()

    def qkv_norm_rotary_cached(self, qkv, *args, **kw):
        self.seen.add(qkv.dtype)
        return CacheOps.qkv_norm_rotary_cached(qkv, *args, **kw)

    def cached_attention(self, q, *args, **kw):
        self.seen.add(q.dtype)
        return CacheOps.cached_attention(q, *args, **kw)


def model(ops=CacheOps, dtype=F32):
    torch.manual_seed(3)
    return AD.Decoder(AD.DecoderConfig(**CFG, use_attnres=False), ops=ops).to(dtype)


def test_a_cache_is_in_the_dtype_of_the_heads():
    m = model()
    assert m.new_cache(1).k.dtype == F32 and m.new_cache(1, dtype=BF).k.dtype == BF
    with torch.autocast("cpu", BF):
        assert m.new_cache(1).k.dtype == BF and m.new_cache(1, dtype=F32).v.dtype == F32
        with torch.autocast("cpu", enabled=False):
            assert m.new_cache(1).k.dtype == F32
    with torch.autocast("cuda", BF):  # another device's
        assert m.new_cache(1).k.dtype == F32
    assert model(dtype=BF).new_cache(1).k.dtype == BF


@pytest.mark.parametrize("autocast,cache_dtype,want", [(True, None, BF), (True, F32, F32), (False, BF, BF), (False, None, F32)])
def test_pieces_in_the_dtype_of_the_cache(autocast, cache_dtype, want):
    noting = Noting()
    m = model(noting)
    idx = torch.randint(0, 50, (2, 16))
    with torch.no_grad():
        exact = m(idx, return_hidden=True)
        with torch.autocast("cpu", BF, enabled=autocast):
            plain = m(idx, return_hidden=True)
            cache = m.new_cache(2, page_size=4, **({} if cache_dtype is None else dict(dtype=cache_dtype)))
            got = torch.cat([m(idx[:, a:b], return_hidden=True, cache=cache) for a, b in ((0, 7), (7, 8), (8, 9), (9, 16))], 1)
    assert noting.seen == {want} and got.dtype == plain.dtype
    if not autocast and want == F32:
        assert torch.allclose(got, exact, atol=2e-5, rtol=1e-5)
    else:
        # a hidden state is of size 1; in each of six sublayers at most eight roundings of half a step of bf16, 2^-8
        assert float((got.float() - exact).abs().max()) <= 6 * 8 / 256


def test_generate():
    m = model()
    idx = torch.randint(0, 50, (2, 6))
    with torch.autocast("cpu", BF):
        assert m.generate(idx, 9, lengths=[6, 4]).shape == (2, 9)
        assert m.generate(idx, 30, budget=8, recent=2, cache=m.new_cache(2, page_size=4, weights=True, spare_tokens=8)).shape == (2, 30)
