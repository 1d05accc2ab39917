"""Paged caches for the tests, and the cache operators in plain 64-bit form, token by token."""

import math

import torch

U = 2.0 ** -24  # half a step of fp32, relative
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Cache:
    """Pages of B sequences in random order, NaN wherever no token is."""

    def __init__(self, g, dtype, K, Dh, S, cached, room, layout="dense", extra=2, device="cuda", fill=float("nan"),
                 weights=False):
        self.K, self.Dh, self.S, self.B = K, Dh, S, len(cached)
        M = max(1, -(-room // S))
        P = self.B * M + extra
        self.k, self.v = (_pool(P, K, S, Dh, dtype, layout, device, fill) for _ in range(2))
        self.table = torch.randperm(P, generator=g)[:self.B * M].view(self.B, M).to(torch.int32).to(device)
        self.cached = torch.tensor(cached, dtype=torch.int32, device=device)
        self.w = None
        if weights:
            self.w = torch.rand((P, K, S), generator=g).to(device)

    def where(self, b, n):
        """(page, slot) of the first n tokens of sequence b"""
        j = torch.arange(n, device=self.k.device)
        return self.table[b].long()[j // self.S], j % self.S

    def put(self, g, lengths, std=1.0):
        """Random tokens in the first `lengths[b]` places of every sequence."""
        for b, n in enumerate(lengths):
            page, slot = self.where(b, n)
            for t in (self.k, self.v):
                t[page, :, slot] = (torch.randn((n, self.K, self.Dh), generator=g) * std).to(t.device).to(t.dtype)

    def get(self, t, b, n):
        """The first n tokens of sequence b, [K, n, ...]"""
        page, slot = self.where(b, n)
        return t[page, :, slot].transpose(0, 1)


def _pool(P, K, S, Dh, dtype, layout, device, fill):
    if layout == "dense":
        return torch.full((P, K, S, Dh), fill, dtype=dtype, device=device)
    if layout == "tokens":          # a page's tokens in their order, all heads of one together
        return torch.full((P, S, K, Dh), fill, dtype=dtype, device=device).transpose(1, 2)
    if layout == "layer":           # one layer's part of a larger tensor
        return torch.full((P, 3, K, S, Dh), fill, dtype=dtype, device=device)[:, 1]
    if layout == "odd":             # rows that start anywhere
        return torch.full((P, K, S, Dh + 3), fill, dtype=dtype, device=device)[..., 1:Dh + 1]
    raise ValueError(layout)


def attend_ref(c, q, cached, fresh, scale, k=None, v=None):
    """(out, bound, p): out [B, H, T, Dh] in 64 bits; bound, how far a kernel may be from it; p[b][h]: [T][n] weights.

    bound: half a step of the dtype of the result, and of sum p |v| the share
      2 d + (n + 16) u + 2^-16 (16 bits: p in two terms, the second the rest of the first, 2^-8 of it at most, and off by
      2^-8 of itself),
      d = (Dh + 8) u scale sum |q k| + 8 u |s|: the fp32 sum of a score, its scaling and the exponential.
    """
    B, H, T, Dh = q.shape
    out = torch.zeros((B, H, T, Dh), dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    ps = {}
    for b in range(B):
        for t in range(T):
            if t >= fresh[b]:
                continue
            n = cached[b] + t + 1
            kk = c.get(c.k if k is None else k, b, n).double()
            vv = c.get(c.v if v is None else v, b, n).double()
            for h in range(H):
                x = q[b, h, t].double()
                kh, vh = kk[h // (H // c.K)], vv[h // (H // c.K)]
                s = (kh * x).sum(-1) * scale
                p = torch.exp(s - s.max())
                p = p / p.sum()
                out[b, h, t] = (p[:, None] * vh).sum(0)
                mag = (kh * x).abs().sum(-1) * abs(scale)
                d = float(((Dh + 8) * U * mag + 8 * U * s.abs()).max())
                share = 2 * d + (n + 16) * U + (0.0 if q.dtype == torch.float32 else 2.0 ** -16)
                bound[b, h, t] = HALF_STEP[q.dtype] * out[b, h, t].abs() * (1 + share) + share * (p[:, None] * vh.abs()).sum(0)
                ps[b, h, t] = (p, share)
    return out, bound, ps


def assert_within(a, e, bound, name=""):
    d = (a.double() - e).abs()
    bad = ~(d <= bound + 1e-30)
    assert not bool(bad.any()), (f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float(d[bad].max()):.3e} where "
                                 f"{float(bound[bad].flatten()[d[bad].argmax()]):.3e} is allowed")


def append_ref(qkv, H, K, sin, cos, positions, eps=2.0 ** -23, qk_norm=True):
    """(heads, bound): rotated query and key heads [B, T, H + K, Dh] in 64 bits; fp32 sums of Dh squares, a root, a
    division, two products and a sum: (Dh + 16) u of |even| + |odd| and half a step of the dtype."""
    B, T, C = qkv.shape
    Dh = C // (H + 2 * K)
    x = qkv.double().view(B, T, H + 2 * K, Dh)[:, :, :H + K]
    if qk_norm:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    s, c = (t.double()[positions][:, :, None] for t in (sin, cos))
    even, odd = x[..., 0::2], x[..., 1::2]
    y = torch.stack([c * even - s * odd, s * even + c * odd], -1).flatten(-2)
    mag = (even.abs() + odd.abs()).repeat_interleave(2, -1)
    return y, HALF_STEP[qkv.dtype] * y.abs() + (Dh + 16) * U * mag * (1 + HALF_STEP[qkv.dtype])


def evict_ref(weights, n, budget, recent):
    """Places kept of n tokens with these weights (a list of floats)."""
    if n <= budget:
        return list(range(n))
    early = n - recent

    def order(j):
        w = weights[j]
        return (1, 0.0, j) if math.isnan(w) else (0, -w, j)

    return sorted(sorted(range(early), key=order)[:budget - recent]) + list(range(early, n))
