"""Workloads of the decoder's sublayer operators, through the drop-in module's public functions.

``rotary`` cases: ``attnres_ops.qkv_norm_rotary`` -- the heads of a fused query / key / value projection, queries and
keys rms-normed per head and rotated by their positions, forward and (``train``) backward into the projection.
``gated`` cases: ``attnres_ops.swiglu_projection`` -- both projections of a gated feed-forward block, the activation and
the product, forward and (``train``) backward into the input and the weight.

A case is a plain dict.  B, T are batch and tokens; H, K, Dh the query heads, key / value heads and head width; D, F
the model width and the hidden width.
"""

from __future__ import annotations

import math
import os
import sys

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


def _rotary(name, **kw):
    # positions: "rows" (token t at position t), "offset" (a chunk behind `start` cached tokens), "each" (one of its
    # own for every token); table: the type of sin / cos (a bf16 model's buffers are bf16)
    c = dict(name=name, family="rotary", B=1, T=1, H=12, K=12, Dh=64, dtype="bf16", table="fp32", positions="rows",
             start=0, train=True)
    c.update(kw)
    return c


def _gated(name, **kw):
    c = dict(name=name, family="gated", B=1, T=1, D=1024, F=4096, dtype="bf16", train=True)
    c.update(kw)
    return c


def listed():
    return [
        # generation with the 12-layer d768 decoder: one new token of 8 sequences of different lengths
        _rotary("rotary_decode", B=8, T=1, positions="each", train=False),
        # a prompt's second chunk, grouped key / value heads, fp16
        _rotary("rotary_prefill_fp16", T=1999, H=16, K=8, Dh=128, dtype="fp16", positions="offset", start=2048,
                train=False),
        # training the 12-layer d768 decoder, all of its buffers in bf16
        _rotary("rotary_train_d768", B=16, T=1024, table="bf16"),
        # training at long sequences with wide heads
        _rotary("rotary_train_long", B=2, T=8192, H=16, K=16, Dh=128),
        # a small fp32 model with a head width that is no power of two, ragged length
        _rotary("rotary_train_fp32", B=3, T=257, H=5, K=5, Dh=40, dtype="fp32"),
        # generation, one sequence: the block reads its weights for one row
        _gated("gated_decode_one", D=768, F=2048, train=False),
        # generation, 40 sequences
        _gated("gated_decode_40", B=40, train=False),
        # a prompt of the 24-layer d1024 decoder, fp16
        _gated("gated_prefill_fp16", T=2000, dtype="fp16", train=False),
        # training the d768 decoder's block on 16384 tokens
        _gated("gated_train_d768", B=16, T=1024, D=768, F=2048),
        # training the published 24-layer d1024 decoder's block on 16384 tokens
        _gated("gated_train_d1024", B=8, T=2048),
        # widths that fill no tile and no 16-byte vector, ragged token count
        _gated("gated_train_ragged", B=3, T=677, D=500, F=1363),
        # a small fp32 model
        _gated("gated_train_fp32", B=2, T=256, D=256, F=688, dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_MOST_VALUES = 2 * 8192 * 3 * 2048          # of rotary_train_long's projection
_MOST_PRODUCTS = 16384 * 1024 * 4096        # of gated_train_d1024


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    tokens = _log_int(rng, 1, 16384)
    B = rng.choice([1, 1, 2, 3, 4, 8, 16])
    T = max(1, tokens // B)
    train = rng.random() < 0.6
    if rng.random() < 0.5:
        K = rng.randint(1, 16)
        H = K * rng.choice([1, 1, 1, 2, 4])
        Dh = rng.choice([32, 64, 64, 96, 128, 128, 256, 2 * rng.randint(4, 100)])
        T = max(1, min(T, _MOST_VALUES // (B * (H + 2 * K) * Dh * (2 if dtype == "fp32" else 1))))
        positions = rng.choice(["rows", "offset", "each"])
        return dict(family="rotary", B=B, T=T, H=H, K=K, Dh=Dh, dtype=dtype, table=rng.choice(["fp32", dtype]),
                    positions=positions, start=rng.randint(1, 4096) if positions == "offset" else 0, train=train)
    D, F = (8 * _log_int(rng, 8, 256) if rng.random() < 0.75 else _log_int(rng, 64, 2048),
            8 * _log_int(rng, 8, 512) if rng.random() < 0.75 else _log_int(rng, 64, 4096))
    most = _MOST_PRODUCTS // (16 if dtype == "fp32" else 1)
    T = max(1, min(T, most // (B * D * F)))
    return dict(family="gated", B=B, T=T, D=D, F=F, dtype=dtype, train=train)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    B, T = case["B"], case["T"]

    def randn(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dt)

    if case["family"] == "gated":
        D, F = case["D"], case["F"]
        # the block's input is a normed row; weights of a trained model's size
        s = dict(case, x=randn(B, T, D), weight=randn(2 * F, D, std=1.5 * D ** -0.5))
        if case["train"]:
            s["grad"] = randn(B, T, F)
            s["x"].requires_grad_(True)
            s["weight"].requires_grad_(True)
        return s
    H, K, Dh = case["H"], case["K"], case["Dh"]
    qkv = torch.randn((B, T, H + 2 * K, Dh), generator=g, device="cuda")
    # heads of different sizes, as projections learn them
    qkv *= torch.exp2(torch.randn((H + 2 * K, 1), generator=g, device="cuda"))
    qkv = qkv.to(dt).view(B, T, (H + 2 * K) * Dh)
    rows = max(4096, case["start"] + T)
    inv_freq = THETA ** (-torch.arange(0, Dh, 2, device="cuda", dtype=torch.float64) / Dh)
    angle = torch.outer(torch.arange(rows, device="cuda", dtype=torch.float64), inv_freq)
    table = DTYPES[case["table"]]
    s = dict(case, qkv=qkv, sin=angle.sin().to(table), cos=angle.cos().to(table))
    s["at"] = {"rows": None, "offset": case["start"]}.get(case["positions"])
    if case["positions"] == "each":
        s["at"] = torch.randint(0, rows, (B, T), generator=g, device="cuda")
    if case["train"]:
        # the upstream gradients, as attention's backward gives them
        s["grads"] = [randn(B, h, T, Dh) for h in (H, K, K)]
        qkv.requires_grad_(True)
    return s


def run(s):
    return (_run_gated if s["family"] == "gated" else _run_rotary)(s)


def _run_gated(s):
    x, weight = s["x"], s["weight"]
    if own:
        h = _ops().swiglu_projection(x, weight)
        if not s["train"]:
            return [h]
        return [h.detach(), *torch.autograd.grad(h, [x, weight], s["grad"])]
    with torch.no_grad():
        dt, (B, T, D) = x.dtype, x.shape
        x = x.reshape(B * T, D).float()
        w = weight.float()
        up, gate = (x @ w.t()).chunk(2, dim=1)
        sig = 1.0 / (1.0 + torch.exp(-gate))
        act = gate * sig
        h = (act * up).to(dt).view(B, T, -1)
        if not s["train"]:
            return [h]
        dh = s["grad"].reshape(B * T, -1).float()
        d = torch.cat([dh * act, dh * up * (sig + act * (1.0 - sig))], dim=1)
        return [h, (d @ w).to(dt).view(B, T, D), (d.t() @ x).to(dt)]


def _angles(s):
    """sin and cos of every token, [B or 1, T, 1, Dh / 2] in the tables' type."""
    at = s["at"]
    if isinstance(at, torch.Tensor):
        return s["sin"][at][:, :, None], s["cos"][at][:, :, None]
    start = at or 0
    return tuple(t[start:start + s["T"]][None, :, None] for t in (s["sin"], s["cos"]))


def _run_rotary(s):
    qkv, B, T, H, K, Dh = s["qkv"], s["B"], s["T"], s["H"], s["K"], s["Dh"]
    if own:
        q, k, v = _ops().qkv_norm_rotary(qkv, H, s["sin"], s["cos"], positions=s["at"], num_kv_heads=K)
        if not s["train"]:
            return [q, k, v]
        (d,) = torch.autograd.grad([q, k, v], [qkv], s["grads"])
        return [q.detach(), k.detach(), v.detach(), d]
    with torch.no_grad():
        dt = qkv.dtype
        heads = qkv.view(B, T, H + 2 * K, Dh)
        x = heads[:, :, :H + K].float()
        sin, cos = (t.float() for t in _angles(s))
        inv = torch.rsqrt((x * x).sum(-1, keepdim=True) / Dh + EPS)
        n = x * inv
        even, odd = n[..., 0::2], n[..., 1::2]
        y = torch.stack([cos * even - sin * odd, sin * even + cos * odd], dim=-1).flatten(-2)
        y = y.to(dt).transpose(1, 2)
        out = [y[:, :H], y[:, H:], heads[:, :, H + K:].transpose(1, 2)]
        if not s["train"]:
            return out
        g = torch.cat(s["grads"][:2], dim=1).transpose(1, 2).float()
        even, odd = g[..., 0::2], g[..., 1::2]
        g = torch.stack([cos * even + sin * odd, cos * odd - sin * even], dim=-1).flatten(-2)
        dx = inv * (g - n * ((g * n).sum(-1, keepdim=True) / Dh))
        d = torch.cat([dx.to(dt), s["grads"][2].transpose(1, 2)], dim=2)
        return [*out, d.reshape(B, T, -1)]


def work(case):
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    n = case["B"] * case["T"]
    if case["family"] == "gated":
        D, F = case["D"], case["F"]
        # x and W read, h written; with training the upstream gradient read, dx and dW written
        values = n * D + 2 * F * D + n * F
        if case["train"]:
            values += n * F + n * D + 2 * F * D
        return {"bytes": values * size, "flops": 4 * n * D * F * (3 if case["train"] else 1)}
    H, K, Dh = case["H"], case["K"], case["Dh"]
    table = torch.finfo(DTYPES[case["table"]]).bits // 8
    rows = n if case["positions"] == "each" else case["T"]
    # queries and keys read and written; with training the three upstream gradients read, the projection's written
    values = 2 * n * (H + K) * Dh + (2 * n * (H + 2 * K) * Dh if case["train"] else 0)
    # norm: a product and a sum each, and the scale; rotation: two products and a sum an element; backward the same
    # again with the norm's correction
    flops = n * (H + K) * Dh * (6 + (11 if case["train"] else 0))
    return {"bytes": values * size + rows * Dh * table + (8 * n if case["positions"] == "each" else 0), "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return (_exact_gated if case["family"] == "gated" else _exact_rotary)(s)


def _exact_gated(s):
    x, w = s["x"].double().flatten(0, 1), s["weight"].double()
    lead, F = s["x"].shape[:2], s["F"]
    u = torch.mm(x, w[:F].t())
    z = torch.mm(x, w[F:].t())
    half = torch.tanh(z / 2)  # logistic(z) = (1 + tanh(z / 2)) / 2
    silu = z * (1 + half) / 2
    h = (u * silu).view(*lead, F)
    if not s["train"]:
        return [h]
    dh = s["grad"].double().flatten(0, 1)
    du = dh * silu
    dz = dh * u * ((1 + half) / 2 + z * (1 - half * half) / 4)
    dx = torch.mm(du, w[:F]) + torch.mm(dz, w[F:])
    return [h, dx.view(s["x"].shape), torch.cat([torch.mm(du.t(), x), torch.mm(dz.t(), x)])]


def _exact_rotary(s):
    B, T, H, K, Dh = s["B"], s["T"], s["H"], s["K"], s["Dh"]
    # pairs as complex numbers: the rotation is a product with cos + i sin
    z = torch.view_as_complex(s["qkv"].detach().double().view(B, T, H + 2 * K, Dh // 2, 2)).transpose(1, 2)
    sin, cos = (t.double().transpose(1, 2) for t in _angles(s))
    turn = torch.complex(cos.contiguous(), sin.contiguous())
    r = torch.sqrt((z.real.square() + z.imag.square()).sum(-1, keepdim=True) / Dh + EPS)
    z, v, unit, r = z[:, :H + K], z[:, H + K:], (z / r)[:, :H + K], r[:, :H + K]

    def real(c):
        return torch.view_as_real(c.contiguous()).flatten(-2)

    y = unit * turn
    out = [real(y[:, :H]), real(y[:, H:]), real(v)]
    if not s["train"]:
        return out
    g = torch.cat(s["grads"][:2], dim=1).double()
    g = torch.view_as_complex(g.view(B, H + K, T, Dh // 2, 2)) * turn.conj()
    along = (g * unit.conj()).real.sum(-1, keepdim=True) / Dh
    d = torch.cat([real((g - unit * along) / r), s["grads"][2].double()], dim=1)
    return [*out, d.transpose(1, 2).reshape(B, T, -1)]
