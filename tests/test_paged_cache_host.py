"""CPU checks of the paged cache's bookkeeping where calls fail, and of what generation refuses before it has done anything."""

import pytest
import torch

import attnres_decoder as AD
from attnres_cache import PagedCache
from test_decoder_cache_host import CFG, CacheOps


def filled(lengths, max_tokens=12, spare=6, **kw):
    g = torch.Generator().manual_seed(5)
    c = PagedCache(2, 2, 4, len(lengths), max_tokens, page_size=4, dtype=torch.float32, device="cpu", weights=True,
                   spare_tokens=spare, **kw)
    for t in (c.k, c.v, c.weights):
        t.copy_(torch.randn(t.shape, generator=g))
    c.reserve(lengths)
    c.advance(lengths)
    return c


class Failing(CacheOps):
    """Raises in the call of the layer given."""

    def __init__(self, layer):
        self.left = layer

    def evict_cached_tokens(self, *args):
        if self.left == 0:
            raise RuntimeError("launch failed")
        self.left -= 1
        return CacheOps.evict_cached_tokens(*args)


@pytest.mark.parametrize("layer", [0, 1])
def test_an_eviction_that_raises_leaves_the_cache_as_it_was(layer):
    c, want = filled([12, 3, 9]), filled([12, 3, 9])
    before = (list(c._free), [list(o) for o in c._owned], c.table.clone(), c.cached.clone(), list(c.lengths))
    with pytest.raises(RuntimeError, match="launch failed"):
        c.evict(Failing(layer), 6, 2)
    assert (c._free, c._owned, c.lengths) == (before[0], before[1], before[4])
    assert torch.equal(c.table, before[2]) and torch.equal(c.cached, before[3])
    # the same call again, as if it were the first
    for a, b in zip(c.evict(CacheOps, 6, 2), want.evict(CacheOps, 6, 2)):
        assert torch.equal(a, b)
    assert torch.equal(c.table, want.table) and torch.equal(c.cached, want.cached) and c.lengths == want.lengths
    for b, n in enumerate(c.lengths):
        j = torch.arange(n)
        page, slot = c.table[b].long()[j // 4], j % 4
        for x, y in ((c.k, want.k), (c.v, want.v), (c.weights, want.weights)):
            assert torch.equal(x[:, page, :, slot], y[:, page, :, slot])


def decoder():
    torch.manual_seed(3)
    return AD.Decoder(AD.DecoderConfig(**CFG), ops=CacheOps)


@pytest.mark.parametrize("weights,budget,recent,error", [
    (False, 8, 2, RuntimeError), (True, 0, 0, ValueError), (True, 8, 9, ValueError), (True, 8, -1, ValueError), (True, -3, 0, ValueError)])
def test_generate_refuses_a_budget_before_its_first_token(weights, budget, recent, error):
    m = decoder()
    idx = torch.randint(0, 50, (2, 6))
    cache = m.new_cache(2, page_size=4, weights=weights, spare_tokens=8)
    with pytest.raises(error):
        m.generate(idx, 3, cache=cache, budget=budget, recent=recent)
    assert cache.lengths == [0, 0] and len(cache._free) == cache.pages
    if weights:
        with pytest.raises(error):
            m.generate(idx, 3, budget=budget, recent=recent)


def test_a_cache_with_less_than_a_page_above_the_budget():
    """It is full before a sequence is a page above its budget: brought back then."""
    m = decoder()
    idx = torch.randint(0, 50, (2, 6))
    cache = m.new_cache(2, 12, page_size=4, weights=True, spare_tokens=10)
    out = m.generate(idx, 20, cache=cache, budget=10, recent=4)
    assert out.shape == (2, 20) and max(cache.lengths) <= 12 and cache.next_positions == [25, 25]
    assert cache.cached.tolist() == cache.lengths
