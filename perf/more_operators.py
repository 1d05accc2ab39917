"""Workloads of the decoder's paged key-value cache, through the drop-in module's public functions.

``append`` cases: ``attnres_ops.qkv_norm_rotary_cached`` -- the heads of the new tokens' projection, queries and keys
normed and rotated at each sequence's own position, keys and values written into their pages.
``attend`` cases: ``attnres_ops.cached_attention`` -- attention of the newest tokens over the pages, with ``weights`` also
what each cached token received of it (the call starts a sum anew: decay 0).
``evict`` cases: ``attnres_ops.evict_cached_tokens`` -- per key / value head the most attended and the last tokens, moved in
their order into other pages.

A case is a plain dict.  B, T are sequences and new tokens of each; H, K, Dh the query heads, key / value heads and head
width; page the tokens of a page; low .. high the tokens that a sequence has in the cache before the call (``spread``:
between the two, else all ``high``).
"""

from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = float(torch.finfo(torch.float32).eps)  # the rms-norms' eps, for every dtype
THETA = 500000.0  # the decoder's rotary base


def _ops():
    pkg = os.path.join(ROOT, "lr-attnres_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import attnres_ops
    return attnres_ops


def _attend(name, **kw):
    c = dict(name=name, family="attend", B=1, T=1, H=12, K=12, Dh=64, page=64, low=0, high=1024, dtype="bf16",
             weights=False)
    c.update(kw)
    return c


def _append(name, **kw):
    # padded: sequences have different numbers of the T new tokens (a batch of prompts); heads: the call hands back the
    # rotated keys and the values too, for attention inside the prompt
    c = dict(name=name, family="append", B=1, T=1, H=12, K=12, Dh=64, page=64, low=0, high=1024, dtype="bf16",
             table="fp32", padded=False, heads=False)
    c.update(kw)
    return c


def _evict(name, **kw):
    c = dict(name=name, family="evict", B=1, K=12, Dh=64, page=64, low=0, high=2048, budget=1024, recent=128,
             dtype="bf16")
    c.update(kw)
    return c


def listed():
    return [
        # generation with the 12-layer d768 decoder: one sequence, early in its answer
        _attend("attend_one", low=300, high=300),
        # the same decoder, 16 sequences of different lengths
        _attend("attend_d768", B=16, low=128, high=2047),
        # long contexts, grouped key / value heads
        _attend("attend_long", B=4, H=16, K=4, Dh=128, low=32768, high=131071),
        # a cache under a budget: attention counts what each token receives; fp16, small pages
        _attend("attend_weights", B=8, H=16, K=8, Dh=128, page=16, low=4096, high=8191, dtype="fp16", weights=True),
        # seven drafted tokens at once
        _attend("attend_drafts", B=4, T=7, H=16, K=4, page=32, low=512, high=4096),
        # a small fp32 model: a head width that is no power of two, pages that end inside tiles, an empty cache among them
        _attend("attend_fp32", B=3, H=5, K=5, Dh=40, page=24, low=0, high=700, dtype="fp32"),
        # a generation step of the d768 decoder, 16 sequences, all of its buffers in bf16
        _append("append_step", B=16, low=128, high=2047, table="bf16"),
        # a batch of prompts of the published d1024 decoder, padded to 2048
        _append("append_prompts", B=8, T=2048, H=16, K=16, low=0, high=0, padded=True, heads=True),
        # chunks of the small fp32 model's prompts behind what is cached
        _append("append_fp32", B=3, T=37, H=5, K=5, Dh=40, page=24, low=0, high=90, dtype="fp32", heads=True),
        # the d768 decoder's layer brought back to 1024 tokens, sequences within it among them
        _evict("evict_d768", B=16, low=900, high=2048),
        # long contexts brought back to 8192 tokens
        _evict("evict_long", B=2, K=8, Dh=128, low=32768, high=65536, budget=8192, recent=1024),
        # the small fp32 model
        _evict("evict_fp32", B=3, K=5, Dh=40, page=24, low=0, high=700, budget=256, recent=32, dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_MOST_CACHED = 4 * 4 * 128 * 2 * 65536      # values of attend_long's keys and values, about
_MOST_NEW = 8 * 2048 * 48 * 64              # values of append_prompts' projection
_MOST_KEPT = 2 * 8 * 8192 * 128             # values of evict_long's kept keys


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    size = 2 if dtype == "fp32" else 1
    page = rng.choice([16, 32, 64, 64, 128, 256, rng.randint(1, 100)])
    B = _log_int(rng, 1, 64)
    K = rng.randint(1, 16)
    Dh = rng.choice([32, 64, 64, 96, 128, 128, 256, 2 * rng.randint(4, 128)])
    family = rng.choice(["attend", "attend", "append", "evict"])
    if family == "attend":
        H = K * rng.choice([1, 1, 2, 4, 8, rng.randint(1, 20)])
        T = rng.choice([1, 1, 1, rng.randint(2, 16)])
        high = min(_log_int(rng, 1, 131072), max(1, _MOST_CACHED // (size * B * K * Dh * 2 * -(-H * T // (K * 16)))))
        low = rng.choice([0, high // 4, high // 2, high])
        return dict(family=family, B=B, T=T, H=H, K=K, Dh=Dh, page=page, low=low, high=high, dtype=dtype,
                    weights=T == 1 and rng.random() < 0.3)
    if family == "append":
        H = K * rng.choice([1, 1, 2, 4])
        T = max(1, min(_log_int(rng, 1, 2048), _MOST_NEW // (size * B * (H + 2 * K) * Dh)))
        high = _log_int(rng, 1, 8192)
        return dict(family=family, B=B, T=T, H=H, K=K, Dh=Dh, page=page, low=rng.choice([0, high // 2, high]), high=high,
                    dtype=dtype, table=rng.choice(["fp32", dtype]), padded=T > 1 and rng.random() < 0.5,
                    heads=rng.random() < 0.5)
    budget = max(1, min(_log_int(rng, 16, 8192), _MOST_KEPT // (size * B * K * Dh)))
    high = min(65536, budget * rng.choice([1, 2, 4]) + rng.randint(0, 100))
    return dict(family=family, B=B, K=K, Dh=Dh, page=page, low=rng.choice([0, high // 2, high]), high=high, budget=budget,
                recent=rng.choice([0, budget // 8, budget // 2, budget]), dtype=dtype)


def _spread(lo, hi, count):
    """`count` whole numbers of lo .. hi, hi among them; the same for the same arguments."""
    r = random.Random(lo * 1000003 + hi * 101 + count)
    return [hi] + [r.randint(lo, hi) for _ in range(count - 1)]


def _fresh(case):
    return _spread(1, case["T"], case["B"]) if case.get("padded") else [case.get("T", 0)] * case["B"]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    B, K, Dh, page = (case[k] for k in ("B", "K", "Dh", "page"))
    T, family = case.get("T", 0), case["family"]

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    per = max(1, -(-(case["high"] + T) // page))           # pages of a sequence
    per_new = -(-case["budget"] // page) if family == "evict" else 0
    pages = B * (per + per_new) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    # pages that were given back and taken again hold what earlier tokens left
    s = dict(case, k=randn(pages, K, page, Dh).to(dt), v=randn(pages, K, page, Dh).to(dt), w=None,
             table=order[:B * per].view(B, per).contiguous(),
             cached=torch.tensor(_spread(case["low"], case["high"], B), dtype=torch.int32, device="cuda"))
    if family == "attend":
        # heads of different sharpness
        s["q"] = (randn(B, case["H"], T, Dh) * torch.exp2(0.5 + randn(case["H"], 1, 1))).to(dt)
        if case["weights"]:
            s["w"] = torch.rand((pages, K, page), generator=g, device="cuda")
    elif family == "append":
        H = case["H"]
        qkv = randn(B, T, H + 2 * K, Dh) * torch.exp2(randn(H + 2 * K, 1))  # heads of different sizes
        s["qkv"] = qkv.to(dt).view(B, T, (H + 2 * K) * Dh)
        rows = max(4096, case["high"] + T)
        inv_freq = THETA ** (-torch.arange(0, Dh, 2, device="cuda", dtype=torch.float64) / Dh)
        angle = torch.outer(torch.arange(rows, device="cuda", dtype=torch.float64), inv_freq)
        s["sin"], s["cos"] = (t.to(DTYPES[case["table"]]) for t in (angle.sin(), angle.cos()))
        s["fresh"] = torch.tensor(_fresh(case), dtype=torch.int32, device="cuda") if case["padded"] else None
    else:
        # sums of attention weights: most tokens get little, a few a lot, some nothing at all
        w = torch.exp(3 * randn(pages, K, page))
        s["w"] = torch.where(torch.rand(w.shape, generator=g, device="cuda") < 0.1, 0.0, w)
        s["new_table"] = order[B * per:B * (per + per_new)].view(B, per_new).contiguous()
    return s


def run(s):
    return {"attend": _run_attend, "append": _run_append, "evict": _run_evict}[s["family"]](s)


def _pages_of(s, at):
    """(page, slot) of the tokens `at` [B, ...] of every sequence, as indices."""
    t, page = s["table"].long(), s["page"]
    return t.gather(1, (at // page).flatten(1)).view(at.shape), at % page


@torch.no_grad()
def _run_attend(s):
    if own:
        o = _ops().cached_attention(s["q"], s["k"], s["v"], s["table"], s["cached"], weights=s["w"],
                                    decay=0.0 if s["weights"] else 1.0)
        return [o, s["w"]] if s["weights"] else [o]
    q, (B, H, T, Dh), K = s["q"], s["q"].shape, s["K"]
    n = s["table"].size(1) * s["page"]
    table = s["table"].long()
    k, v = (t[table].transpose(1, 2).reshape(B, K, n, Dh).float() for t in (s["k"], s["v"]))
    x = torch.matmul(q.float().view(B, K, H // K * T, Dh), k.transpose(2, 3)).view(B, K, H // K, T, n) * Dh ** -0.5
    last = s["cached"].view(B, 1) + torch.arange(T, device="cuda")
    at = torch.arange(n, device="cuda")
    seen = at <= last.view(B, 1, 1, T, 1)
    x = torch.where(seen, x, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, K, H // K * T, n), v).view(B, H, T, Dh).to(q.dtype)
    if not s["weights"]:
        return [o]
    page, slot = _pages_of(s, at.expand(B, n))
    old = s["w"][page, :, slot]
    s["w"][page, :, slot] = torch.where((at <= last)[..., None], p.sum((2, 3)).transpose(1, 2), old)
    return [o, s["w"]]


def _angles(s):
    """sin and cos of every new token, [B, T, 1, Dh / 2]."""
    at = s["cached"].view(-1, 1).long() + torch.arange(s["T"], device="cuda")
    return s["sin"][at][:, :, None], s["cos"][at][:, :, None]


@torch.no_grad()
def _run_append(s):
    qkv, B, T, H, K, Dh = (s[k] for k in ("qkv", "B", "T", "H", "K", "Dh"))
    if own:
        out = _ops().qkv_norm_rotary_cached(qkv, H, s["sin"], s["cos"], s["k"], s["v"], s["table"], s["cached"],
                                            fresh=s["fresh"], return_heads=s["heads"])
        return [*(out if s["heads"] else [out]), s["k"], s["v"]]
    heads = qkv.view(B, T, H + 2 * K, Dh)
    x = heads[:, :, :H + K].float()
    sin, cos = (t.float() for t in _angles(s))
    n = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / Dh + EPS)
    even, odd = n[..., 0::2], n[..., 1::2]
    y = torch.stack([cos * even - sin * odd, sin * even + cos * odd], dim=-1).flatten(-2)
    t = torch.arange(T, device="cuda")
    real = (t < s["fresh"].view(B, 1) if s["padded"] else (t >= 0).expand(B, T))[..., None, None]
    y = torch.where(real, y, 0.0).to(qkv.dtype)
    page, slot = _pages_of(s, s["cached"].view(B, 1).long() + t)
    s["k"][page, :, slot] = torch.where(real, y[:, :, H:], s["k"][page, :, slot])
    s["v"][page, :, slot] = torch.where(real, heads[:, :, H + K:], s["v"][page, :, slot])
    y, v = y.transpose(1, 2), heads[:, :, H + K:].transpose(1, 2)
    return [y[:, :H], *([y[:, H:], v] if s["heads"] else []), s["k"], s["v"]]


@torch.no_grad()
def _run_evict(s):
    if own:
        kept, left = _ops().evict_cached_tokens(s["k"], s["v"], s["w"], s["table"], s["cached"], s["new_table"],
                                                s["budget"], s["recent"])
        return [kept, left, s["k"], s["v"], s["w"]]
    B, K, page, budget = s["B"], s["K"], s["page"], s["budget"]
    n = s["table"].size(1) * page
    w = s["w"][s["table"].long()].transpose(1, 2).reshape(B, K, n)
    at, have = torch.arange(n, device="cuda"), s["cached"].view(B, 1, 1)
    w = torch.where(at >= have, -math.inf, torch.where(at >= have - s["recent"], math.inf, w))
    first = torch.sort(w, dim=-1, descending=True, stable=True)[1][..., :budget]
    first = torch.sort(torch.where(first < have, first, n), dim=-1)[0]
    if n < budget:
        first = torch.cat([first, first.new_full((B, K, budget - n), n)], dim=-1)
    kept = torch.where(first < n, first, -1).to(torch.int32)
    src, slot = _pages_of(s, first.clamp(max=n - 1))
    to = torch.arange(budget, device="cuda")
    page_to, slot_to = s["new_table"].long()[:, None, to // page], (to % page).expand(B, K, budget)
    head = torch.arange(K, device="cuda").view(1, K, 1)
    real = first < n
    for t in (s["k"], s["v"], s["w"]):
        mask = real if t.dim() == 3 else real[..., None]
        t[page_to, head, slot_to] = torch.where(mask, t[src, head, slot], t[page_to, head, slot_to])
    return [kept, s["cached"].clamp(max=budget), s["k"], s["v"], s["w"]]


def work(case):
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    B, K, Dh = case["B"], case["K"], case["Dh"]
    cached = _spread(case["low"], case["high"], B)
    if case["family"] == "attend":
        H, T = case["H"], case["T"]
        tokens = sum(cached) + B * T
        seen = sum(T * n + T * (T + 1) // 2 for n in cached)
        # keys and values read, queries read, the output written; a sum written for every token's key / value heads
        return {"bytes": (2 * tokens * K + 2 * B * T * H) * Dh * size + (4 * tokens * K if case["weights"] else 0),
                "flops": 4 * seen * H * Dh}
    if case["family"] == "append":
        H, new = case["H"], sum(_fresh(case))
        table = torch.finfo(DTYPES[case["table"]]).bits // 8
        # the projection read, queries, keys and values written; rotated keys once more where they are handed back
        return {"bytes": new * ((2 * H + 4 * K + (K if case["heads"] else 0)) * Dh * size + Dh * table),
                "flops": 6 * new * (H + K) * Dh}
    kept = sum(min(n, case["budget"]) for n in cached)
    # every token's weight read, what is kept read and written, with its weight and its place
    return {"bytes": sum(cached) * K * 4 + kept * K * (4 * Dh * size + 8), "flops": sum(cached) * K}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attend": _exact_attend, "append": _exact_append, "evict": _exact_evict}[s["family"]](s)


def _exact_attend(s):
    q, (B, H, T, Dh), K = s["q"], s["q"].shape, s["K"]
    out = torch.empty((B, H, T, Dh), dtype=torch.float64, device="cuda")
    w = None if s["w"] is None else s["w"].double()
    for b, have in enumerate(s["cached"].tolist()):
        pages = s["table"][b, :-(-(have + T) // s["page"])].long()
        for h in range(K):  # a key / value head's tokens in their order
            k, v = (t[pages, h].reshape(-1, Dh)[:have + T].double() for t in (s["k"], s["v"]))
            for t in range(T):
                rows = q[b, h * (H // K):(h + 1) * (H // K), t].double()
                x = torch.mm(rows, k[:have + t + 1].t()) / math.sqrt(Dh)
                p = torch.softmax(x, dim=-1)
                out[b, h * (H // K):(h + 1) * (H // K), t] = torch.mm(p, v[:have + t + 1])
                if w is not None:
                    flat = w[pages, h].reshape(-1)
                    flat[:have + 1] = p.sum(0)
                    w[pages, h] = flat.view(len(pages), -1)
    return [out] if w is None else [out, w]


def _exact_append(s):
    qkv, B, T, H, K, Dh = (s[k] for k in ("qkv", "B", "T", "H", "K", "Dh"))
    # pairs as complex numbers: the rotation is a product with cos + i sin
    z = torch.view_as_complex(qkv.double().view(B, T, H + 2 * K, Dh // 2, 2))
    sin, cos = _angles(s)
    r = torch.sqrt((z.real.square() + z.imag.square()).sum(-1, keepdim=True) / Dh + EPS)
    y = torch.view_as_real(z[:, :, :H + K] / r[:, :, :H + K] * torch.complex(cos.double(), sin.double())).flatten(-2)
    v = qkv.view(B, T, H + 2 * K, Dh)[:, :, H + K:].double()
    k_pages, v_pages = s["k"].double(), s["v"].double()
    table, cached = s["table"].tolist(), s["cached"].tolist()
    for b, new in enumerate(_fresh(s)):
        y[b, new:] = 0
        places = [divmod(cached[b] + t, s["page"]) for t in range(new)]
        page = torch.tensor([table[b][p] for p, _ in places], device="cuda")
        slot = torch.tensor([i for _, i in places], device="cuda")
        k_pages[page, :, slot] = y[b, :new, H:]
        v_pages[page, :, slot] = v[b, :new]
    y = y.transpose(1, 2)
    return [y[:, :H], *([y[:, H:], v.transpose(1, 2)] if s["heads"] else []), k_pages, v_pages]


def _exact_evict(s):
    B, K, page, budget, recent = (s[k] for k in ("B", "K", "page", "budget", "recent"))
    pools = [t.double().cpu().numpy() for t in (s["k"], s["v"], s["w"])]
    old = pools[2].copy()
    table, new, cached = (s[k].cpu().numpy() for k in ("table", "new_table", "cached"))
    kept = np.full((B, K, budget), -1, dtype=np.int32)
    source = [p.copy() for p in pools[:2]]
    for b, h in np.ndindex(B, K):
        have = int(cached[b])
        w = old[table[b], h].reshape(-1)[:have]
        keep = np.arange(have)
        if have > budget:
            early = np.lexsort((np.arange(have - recent), -w[:have - recent]))[:budget - recent]
            keep = np.sort(np.concatenate([early, np.arange(have - recent, have)]))
        kept[b, h, :len(keep)] = keep
        i = np.arange(len(keep))
        at, to = (table[b][keep // page], h, keep % page), (new[b][i // page], h, i % page)
        for p, o in zip(pools, [*source, old]):
            p[to] = o[at]
    return [torch.from_numpy(kept), torch.from_numpy(np.minimum(cached, budget)), *map(torch.from_numpy, pools)]
