"""CPU checks of generation with a paged cache, the oracle standing in for the kernels: a decoder fed its tokens piece by
piece gives the hidden states of one pass over all of them; pages are handed out, moved and given back; refusals."""

import pytest
import torch

import attnres_decoder as AD
from attnres_cache import PagedCache
from decoder_util import OracleOps
from oracle import attnres_oracle as O

CFG = dict(n_layer=3, n_head=2, n_embd=32, mlp_hidden_dim=40, vocab_size=50, block_size=48, attnres_num_blocks=2, lrid_rank=8,
           attn_res_query_init="normal", init_std=0.1)


class CacheOps(OracleOps):
    qkv_norm_rotary_cached = staticmethod(O.qkv_norm_rotary_cached_ref)
    cached_attention = staticmethod(O.cached_attention_ref)
    evict_cached_tokens = staticmethod(O.evict_cached_tokens_ref)


def model(**kw):
    torch.manual_seed(3)
    return AD.Decoder(AD.DecoderConfig(**{**CFG, **kw}), ops=CacheOps)


def cache_for(m, batch, page_size=4, **kw):
    return m.new_cache(batch, page_size=page_size, **kw)


@pytest.mark.parametrize("kw", [dict(), dict(use_attnres=False), dict(norm_pos="both"), dict(qk_norm=False),
                                dict(weight_tying=True, attnres_training_torch_phase2=False)])
@pytest.mark.parametrize("pieces", [[20], [1] * 20, [7, 1, 1, 6, 5], [1, 19]])
def test_pieces_of_a_sequence(kw, pieces):
    m = model(**kw)
    idx = torch.randint(0, 50, (3, 20))
    with torch.no_grad():
        want = m(idx)
        cache, got, at = cache_for(m, 3), [], 0
        for n in pieces:
            got.append(m(idx[:, at:at + n], cache=cache))
            at += n
    # (fp32: the same sums in another order)
    assert torch.allclose(torch.cat(got, 1), want, atol=2e-5, rtol=1e-5)
    assert cache.lengths == [20] * 3 == cache.cached.tolist() == cache.positions.tolist()


def test_padded_prompts_and_steps():
    m = model()
    lengths = [9, 1, 14]
    idx = torch.randint(0, 50, (3, 14))
    more = torch.randint(0, 50, (3, 3))
    with torch.no_grad():
        cache = cache_for(m, 3)
        first = m(idx, cache=cache, fresh=lengths)
        assert cache.lengths == lengths
        # a sequence that takes no part in a step
        second = m(more[:, :2], cache=cache, fresh=[2, 0, 1])
        third = m(more[:, 2:], cache=cache)
        for b, (n, s) in enumerate(zip(lengths, (2, 0, 1))):
            own = torch.cat([idx[b, :n], more[b, :s], more[b, 2:]])[None]
            want = m(own)[0]
            got = torch.cat([first[b, :n], second[b, :s], third[b]])
            assert torch.allclose(got, want, atol=2e-5, rtol=1e-5)
    assert cache.cached.tolist() == cache.lengths == [12, 2, 16]


def test_generate_is_the_largest_logit_of_each_prefix():
    m = model()
    idx = torch.randint(0, 50, (2, 6))
    got = m.generate(idx, 9, lengths=[6, 4])
    for b, n in enumerate((6, 4)):
        seq = idx[b, :n].tolist()
        for t in range(9):
            with torch.no_grad():
                seq.append(int(m(torch.tensor([seq]))[0, -1].argmax()))
        assert got[b].tolist() == seq[n:]
    picked = m.generate(idx, 3, pick=lambda logits: torch.full((logits.size(0),), 7))
    assert picked.tolist() == [[7, 7, 7]] * 2


def test_generate_within_a_budget():
    m = model()
    idx = torch.randint(0, 50, (2, 10))
    cache = cache_for(m, 2, weights=True, spare_tokens=8)
    out = m.generate(idx, 20, cache=cache, budget=8, recent=4)
    assert out.shape == (2, 20)
    assert max(cache.lengths) < 8 + cache.page_size and cache.next_positions == [29, 29] == cache.positions.tolist()
    assert cache.cached.tolist() == cache.lengths
    # one that is never reached changes nothing
    same = m.generate(idx, 20, cache=cache_for(m, 2, weights=True), budget=40)
    assert torch.equal(same, m.generate(idx, 20))


def test_pages():
    c = PagedCache(2, 1, 4, 3, 10, page_size=4, dtype=torch.float32, device="cpu", pages=6)
    assert c.table.shape == (3, 3) and c.pages_in_use() == 1
    c.reserve([4, 5, 0])
    assert (c.table >= 0).sum(1).tolist() == [1, 2, 0] and c.pages_in_use() == 2
    c.advance([4, 5, 0])
    before = c.table.clone()
    with pytest.raises(RuntimeError, match="needed"):
        c.reserve([5, 5, 5])
    with pytest.raises(RuntimeError, match="max_tokens"):
        c.reserve([0, 0, 11])
    assert torch.equal(c.table, before)
    c.reserve([0, 0, 8])
    used = c.table[c.table >= 0].tolist()
    assert len(set(used)) == len(used) == 5
    with pytest.raises(RuntimeError, match="reserve"):
        c.advance([1, 0, 0])
    with pytest.raises(ValueError):
        c.advance([1, 0])
    with pytest.raises(ValueError):
        c.reserve(-1)
    c.drop(1)
    assert c.lengths == [4, 0, 0] and (c.table[1] < 0).all() and c.cached.tolist() == [4, 0, 0]
    c.reserve([0, 9, 0])
    used = c.table[c.table >= 0].tolist()
    assert len(set(used)) == len(used) == 6
    c.replayed([0, 2, 1])
    assert c.lengths == [4, 2, 1] and c.cached.tolist() == [4, 0, 0]


def test_evict_moves_the_long_sequences_only():
    g = torch.Generator().manual_seed(5)
    c = PagedCache(2, 2, 4, 3, 12, page_size=4, dtype=torch.float32, device="cpu", weights=True, spare_tokens=6)
    for t in (c.k, c.v, c.weights):
        t.copy_(torch.randn(t.shape, generator=g))
    c.reserve([12, 3, 9])
    c.advance([12, 3, 9])
    before, row = c.k.clone(), c.table[1].clone()
    old = c.table.clone()
    kept = c.evict(CacheOps, 6, 2)
    assert len(kept) == 2 and c.lengths == [6, 3, 6] == c.cached.tolist() and c.positions.tolist() == [12, 3, 9]
    assert torch.equal(c.table[1], row) and c.k.size(0) == 2
    for i, k in enumerate(kept):
        for b in (0, 2):
            for h in range(2):
                for j, src in enumerate(k[b, h].tolist()):
                    assert torch.equal(c.k[i, c.table[b, j // 4], h, j % 4], before[i, old[b, src // 4], h, src % 4])
    used = c.table[c.table >= 0].tolist()
    assert len(set(used)) == len(used) and len(c._free) + len(used) == c.pages
    assert c.evict(CacheOps, 6, 2) == []
    with pytest.raises(ValueError):
        c.evict(CacheOps, 6, 7)
    with pytest.raises(RuntimeError, match="weights"):
        PagedCache(1, 1, 4, 1, 8, dtype=torch.float32, device="cpu").evict(CacheOps, 4)
    full = PagedCache(1, 1, 4, 1, 8, page_size=4, dtype=torch.float32, device="cpu", weights=True)
    full.reserve(8)
    full.advance(8)
    with pytest.raises(RuntimeError, match="free"):
        full.evict(CacheOps, 4)
    assert full.lengths == [8]


def test_refusals():
    m = model()
    idx = torch.randint(0, 50, (2, 6))
    with torch.no_grad():
        with pytest.raises(ValueError, match="sequences"):
            m(idx, cache=cache_for(m, 3))
        with pytest.raises(ValueError, match="fresh"):
            m(idx, cache=cache_for(m, 2), fresh=[7, 1])
        with pytest.raises(ValueError, match="fresh"):
            m(idx, cache=cache_for(m, 2), fresh=[1])
        cache = cache_for(m, 2)
        for _ in range(8):
            m(idx, cache=cache)
        with pytest.raises(ValueError, match="block_size"):
            m(idx, cache=cache)
        assert cache.lengths == [48, 48]
    with pytest.raises(ValueError, match="block_size"):
        m.generate(idx, 44)
    assert m.generate(idx, 43).shape == (2, 43)
    with pytest.raises(ValueError, match="lengths"):
        m.generate(idx, 2, lengths=[0, 3])
    m.transformer.layers[1].attn.rope = torch.nn.Identity()
    with pytest.raises(NotImplementedError, match="rope"):
        m.generate(idx, 2)
    with pytest.raises(ValueError):
        PagedCache(1, 1, 4, 0, 8)
