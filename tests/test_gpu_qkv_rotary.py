"""Heads of a fused projection: per-head rms-norm and rotary positions (qkv_norm_rotary), forward and backward.

Against 64-bit closed forms, element by element.  Tolerances (u = 2^-24, r = eps / 2 of the dtype): everything is computed
in fp32 and rounded once.  The sum of squares passes at most 8 or 16 additions in a lane and 6 across lanes, so that 1 /
rms is within (22 / 2 + 3) u, a product and a rotated pair add 3 u of the pair's length p = |(even, odd)| / rms: 20 u p in
all.  Backward: the pair of g = R^T dy within 3 u, <g, n> within 30 u |g| |n| (Cauchy), 1 / rms as before: 40 u (pair of g
+ |g| |n| |n_i| / Dh) / rms.
"""

import pytest
import torch

import _attnres_hip as H
import attnres_ops as ops

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
EPS = float(torch.finfo(F32).eps)


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    H.load()
    H.native()


def _tables(rows, Dh, dtype=F32):
    inv = 10000.0 ** (-torch.arange(0, Dh, 2, device="cuda", dtype=torch.float64) / Dh)
    a = torch.outer(torch.arange(rows, device="cuda", dtype=torch.float64), inv)
    return a.sin().to(dtype), a.cos().to(dtype)


def _inputs(B, T, Hq, K, Dh, dtype, seed=0, std=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed + B * 1000 + T * 10 + Hq + Dh)
    rn = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    return rn(B, T, (Hq + 2 * K) * Dh) * std, [rn(B, n, T, Dh) for n in (Hq, K, K)]


def _pairs(t):
    return torch.view_as_complex(t.double().contiguous().view(*t.shape[:-1], t.size(-1) // 2, 2))


def _flat(c):
    return torch.view_as_real(c).flatten(-2)


def _both(t):
    return t.repeat_interleave(2, dim=-1)


def _reference(qkv, sin, cos, at, Hq, K, grads, norm=True):
    """q, k, v, dqkv in 64 bits and the tolerances without the final rounding."""
    B, T, C = qkv.shape
    Dh = C // (Hq + 2 * K)
    heads = qkv.view(B, T, Hq + 2 * K, Dh).transpose(1, 2)
    x, v = _pairs(heads[:, :Hq + K]), heads[:, Hq + K:]
    turn = torch.complex(cos.double()[at], sin.double()[at]).unsqueeze(1)  # [B, 1, T, Dh / 2]
    rms = ((x.abs() ** 2).sum(-1, keepdim=True) / Dh + EPS).sqrt() if norm else torch.ones_like(x.real[..., :1])
    n = x / rms
    y = n * turn
    g = _pairs(torch.cat(grads[:2], 1)) * turn.conj()
    along = (g * n.conj()).real.sum(-1, keepdim=True) / Dh if norm else 0.0
    dx = (g - n * along) / rms
    ty = 20 * U * _both(n.abs() * turn.abs().clamp_min(1.0))
    gn = g.abs().square().sum(-1, keepdim=True).sqrt() * n.abs().square().sum(-1, keepdim=True).sqrt() / Dh
    tx = 40 * U * (_both(g.abs()) + (gn * _both(n.abs()) if norm else 0.0)) / rms
    d = torch.cat([_flat(dx), grads[2].double()], 1).transpose(1, 2).reshape(B, T, C)
    td = torch.cat([tx, torch.zeros_like(v, dtype=torch.float64)], 1).transpose(1, 2).reshape(B, T, C)
    y = _flat(y)
    return (y[:, :Hq], y[:, Hq:], v, d), (ty[:, :Hq], ty[:, Hq:], torch.zeros_like(v, dtype=torch.float64), td)


def _call(qkv, Hq, K, sin, cos, grads, **kw):
    qkv = qkv.detach().requires_grad_(True)
    q, k, v = ops.qkv_norm_rotary(qkv, Hq, sin, cos, num_kv_heads=K, **kw)
    (d,) = torch.autograd.grad([q, k, v], [qkv], grads)
    return q.detach(), k.detach(), v.detach(), d


def _compare(got, want, tol, dtype):
    r = torch.finfo(dtype).eps / 2
    for name, a, e, t in zip("qkvd", got, want, tol):
        assert a.shape == e.shape and a.dtype == dtype
        off = (a.double() - e.double()).abs()
        lim = r * e.double().abs() + (1 + r) * t.double() + float(torch.finfo(dtype).tiny)
        assert not bool((off > lim).any()), (name, float((off / lim).max()))


def _check(B, T, Hq, K, Dh, dtype, table=F32, at=None, norm=True, std=3.0):
    qkv, grads = _inputs(B, T, Hq, K, Dh, dtype, std=std)
    rows = T + 50
    sin, cos = _tables(rows, Dh, table)
    if at is None:
        idx = torch.arange(T, device="cuda").expand(B, T)
    elif isinstance(at, int):
        idx = at + torch.arange(T, device="cuda").expand(B, T)
    else:
        at = torch.randint(0, rows, (B, T) if at == "each" else (T,), device="cuda",
                           generator=torch.Generator(device="cuda").manual_seed(7))
        idx = at.expand(B, T)
    got = _call(qkv, Hq, K, sin, cos, grads, positions=at, qk_norm=norm)
    want, tol = _reference(qkv, sin, cos, idx, Hq, K, grads, norm)
    _compare(got, want, tol, dtype)
    with torch.no_grad():  # the call without a gradient gives the same
        again = ops.qkv_norm_rotary(qkv, Hq, sin, cos, positions=at, num_kv_heads=K, qk_norm=norm)
    assert all(torch.equal(a, b) for a, b in zip(again, got))


@pytest.mark.parametrize("dtype,table", [(BF, F32), (BF, BF), (FP, F32), (FP, FP), (F32, F32)])
@pytest.mark.parametrize("Dh", [2, 4, 6, 8, 16, 32, 34, 40, 64, 68, 96, 128, 130, 198, 200, 256, 258, 264, 512, 1022, 1024])
def test_head_widths(Dh, dtype, table):
    _check(2, 5, 3, 3, Dh, dtype, table)


@pytest.mark.parametrize("Hq,K", [(1, 1), (2, 1), (5, 5), (8, 2), (12, 12), (20, 4), (33, 11), (7, 13)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_head_counts(Hq, K, dtype):
    _check(2, 7, Hq, K, 64, dtype)
    _check(1, 3, Hq, K, 128, dtype)


@pytest.mark.parametrize("B,T", [(1, 1), (8, 1), (1, 2), (3, 257), (2, 1024)])
@pytest.mark.parametrize("at", [None, 3, "row", "each"])
def test_lengths_and_positions(B, T, at):
    _check(B, T, 4, 2, 64, BF, at=at)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_without_norm_and_small_rows(dtype):
    _check(2, 9, 4, 4, 64, dtype, norm=False)
    # rows near and below sqrt(eps): the norm's eps counts (fp16 values are held from 2^-24)
    _check(2, 9, 4, 4, 64, dtype, std=2e-4)


def test_long_table_offsets():
    """Rows of a projection whose last elements lie beyond 2^31 elements: 64-bit offsets."""
    B, T, Hq, K, Dh = 1, 3, 2, 1, 64
    C, stride = (Hq + 2 * K) * Dh, 2 ** 30 + 64
    big = torch.empty((2 * stride + C,), device="cuda", dtype=BF)
    qkv = big.as_strided((B, T, C), (0, stride, 1))
    small, grads = _inputs(B, T, Hq, K, Dh, BF)
    qkv.copy_(small)
    sin, cos = _tables(8, Dh)
    a = ops.qkv_norm_rotary(qkv, Hq, sin, cos, num_kv_heads=K)
    b = ops.qkv_norm_rotary(small, Hq, sin, cos, num_kv_heads=K)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("pad,offset", [(8, 0), (8, 8), (4, 4), (2, 0), (3, 1)])
def test_strided_projections_and_gradients(pad, offset, dtype):
    B, T, Hq, K, Dh = 2, 6, 4, 2, 64
    qkv, grads = _inputs(B, T, Hq, K, Dh, dtype)
    sin, cos = _tables(T, Dh)
    ref = _call(qkv, Hq, K, sin, cos, grads)
    C = qkv.size(-1)
    big = torch.full((B, T + 1, C + pad), float("nan"), device="cuda", dtype=dtype)
    view = big[:, :T, offset:offset + C]
    view.copy_(qkv)
    strided = []
    for g in grads:  # [B, T, heads, Dh + pad] memory, as attention's backward may give them
        m = torch.full((B, T, g.size(1), Dh + pad), float("nan"), device="cuda", dtype=dtype)
        m[..., offset:offset + Dh] = g.transpose(1, 2)
        strided.append(m[..., offset:offset + Dh].transpose(1, 2))
    got = _call(view, Hq, K, sin, cos, strided)
    # (another kernel sums a head's squares in another order: one rounding apart)
    for a, e in zip(got, ref):
        assert float((a.double() - e.double()).abs().max()) <= torch.finfo(dtype).eps * float(e.abs().max())
    # a last dimension that is not dense is copied
    wide = torch.stack([qkv, qkv], dim=-1).flatten(-2)[..., ::2]
    got = _call(wide, Hq, K, sin, cos, [torch.stack([g, g], -1).flatten(-2)[..., ::2] for g in grads])
    assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_missing_and_expanded_gradients():
    B, T, Hq, K, Dh = 2, 5, 4, 2, 64
    qkv, grads = _inputs(B, T, Hq, K, Dh, BF)
    sin, cos = _tables(T, Dh)
    for missing in range(3):
        x = qkv.clone().requires_grad_(True)
        out = ops.qkv_norm_rotary(x, Hq, sin, cos, num_kv_heads=K)
        keep = [i for i in range(3) if i != missing]
        (d,) = torch.autograd.grad([out[i] for i in keep], [x], [grads[i] for i in keep])
        zeros = [torch.zeros_like(g) if i == missing else g for i, g in enumerate(grads)]
        assert torch.equal(d, _call(qkv, Hq, K, sin, cos, zeros)[3])
    one = [torch.ones((), device="cuda", dtype=BF).expand_as(g) for g in grads]
    a, b = _call(qkv, Hq, K, sin, cos, one), _call(qkv, Hq, K, sin, cos, [g.contiguous() for g in one])
    assert torch.equal(a[3], b[3])


def test_positions_outside_the_table_show_as_nan():
    B, T, Hq, K, Dh = 2, 6, 4, 2, 64
    qkv, grads = _inputs(B, T, Hq, K, Dh, BF)
    sin, cos = _tables(T, Dh)
    at = torch.arange(T, device="cuda").expand(B, T).clone()
    ref = _call(qkv, Hq, K, sin, cos, grads, positions=at)
    at[0, 2], at[1, 5] = T, -1
    for w in (64, 1):  # the vector kernels, and the general one (tables that start off a vector)
        s2, c2 = sin, cos
        if w == 1:
            s2, c2 = (torch.cat([t.new_zeros(1), t.flatten()])[1:].view(T, Dh // 2) for t in (sin, cos))
        q, k, v, d = _call(qkv, Hq, K, s2, c2, grads, positions=at)
        bad = [(0, 2), (1, 5)]
        for b in range(B):
            for t in range(T):
                n_rot = (Hq + K) * Dh
                if (b, t) in bad:
                    assert bool(q[b, :, t].isnan().all()) and bool(k[b, :, t].isnan().all())
                    assert bool(d[b, t, :n_rot].isnan().all()) and torch.equal(d[b, t, n_rot:], ref[3][b, t, n_rot:])
                elif w == 64:
                    assert torch.equal(q[b, :, t], ref[0][b, :, t]) and torch.equal(d[b, t], ref[3][b, t])


def test_nan_and_infinities_stay_in_their_heads():
    B, T, Hq, K, Dh = 1, 4, 4, 2, 64
    qkv, grads = _inputs(B, T, Hq, K, Dh, BF)
    sin, cos = _tables(T, Dh)
    ref = _call(qkv, Hq, K, sin, cos, grads)
    bad = qkv.clone()
    bad[0, 1, 2 * Dh + 3] = float("inf")   # query head 2 of token 1
    bad[0, 2, Hq * Dh] = float("nan")      # key head 0 of token 2
    q, k, v, d = _call(bad, Hq, K, sin, cos, grads)
    same_q, same_k = torch.ones((Hq, T), dtype=bool), torch.ones((K, T), dtype=bool)
    same_q[2, 1] = same_k[0, 2] = False
    for a, e, m in ((q, ref[0], same_q), (k, ref[1], same_k)):
        m = m.cuda()
        assert torch.equal(a[0][m], e[0][m]) and bool((a[0][~m].isnan()).any())


def test_zero_rows_empty_inputs_and_views():
    sin, cos = _tables(4, 64)
    x = torch.zeros((1, 4, 3 * 2 * 64), device="cuda", dtype=BF, requires_grad=True)
    q, k, v = ops.qkv_norm_rotary(x, 2, sin, cos)
    assert float(q.abs().max()) == 0.0 and v.data_ptr() == x.data_ptr() + 4 * 64 * 2
    (q.float().sum() + k.float().sum()).backward()
    assert bool(x.grad.isfinite().all())
    e = torch.zeros((0, 4, 384), device="cuda", dtype=BF, requires_grad=True)
    q, k, v = ops.qkv_norm_rotary(e, 2, sin, cos)
    assert q.shape == (0, 2, 4, 64) and v.shape == (0, 2, 4, 64)
    (q.sum() + k.sum() + v.sum()).backward()
    assert e.grad.shape == e.shape
    e = torch.zeros((3, 0, 384), device="cuda", dtype=BF)
    assert ops.qkv_norm_rotary(e, 2, sin, cos)[1].shape == (3, 2, 0, 64)


def test_other_integer_positions_and_table_shapes():
    B, T, Hq, K, Dh = 2, 6, 4, 2, 64
    qkv, _ = _inputs(B, T, Hq, K, Dh, BF)
    sin, cos = _tables(16, Dh)
    at = torch.randint(0, 16, (B, T), device="cuda")
    ref = ops.qkv_norm_rotary(qkv, Hq, sin, cos, positions=at, num_kv_heads=K)
    for t in (torch.int32, torch.int16, torch.uint8):
        got = ops.qkv_norm_rotary(qkv, Hq, sin, cos, positions=at.to(t), num_kv_heads=K)
        assert all(torch.equal(a, b) for a, b in zip(ref, got))
    got = ops.qkv_norm_rotary(qkv, Hq, sin[None, None], cos[None, None], positions=at, num_kv_heads=K)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    wide = at.t().contiguous().t()  # strided positions
    got = ops.qkv_norm_rotary(qkv, Hq, sin, cos, positions=wide, num_kv_heads=K)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    # tables of different types, or strided, are taken in fp32, dense
    s2 = torch.cat([sin, sin], 1)[:, :Dh // 2]
    got = ops.qkv_norm_rotary(qkv, Hq, s2, cos.double(), positions=at, num_kv_heads=K)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))


def test_second_order_streams_and_hooks():
    B, T, Hq, K, Dh = 2, 33, 4, 2, 64
    qkv, grads = _inputs(B, T, Hq, K, Dh, BF)
    sin, cos = _tables(T, Dh)
    ref = _call(qkv, Hq, K, sin, cos, grads)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _call(qkv, Hq, K, sin, cos, grads)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)):
        got = _call(qkv, Hq, K, sin, cos, grads)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    x = qkv.clone().requires_grad_(True)
    q, _, _ = ops.qkv_norm_rotary(x, Hq, sin, cos, num_kv_heads=K)
    (d,) = torch.autograd.grad(q, x, grads[0].clone().requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError, match="twice|once_differentiable"):
        d.sum().backward()


def test_difference_quotients():
    """Against central differences in fp32: third-order term and rounding over the step below 1e-3 of the sizes."""
    B, T, Hq, K, Dh = 1, 3, 2, 1, 16
    qkv, grads = _inputs(B, T, Hq, K, Dh, F32, std=1.0)
    sin, cos = _tables(T, Dh)
    d = _call(qkv, Hq, K, sin, cos, grads)[3]
    e = torch.randn(qkv.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))

    def f(s):
        out = ops.qkv_norm_rotary(qkv + s * e, Hq, sin, cos, num_kv_heads=K)
        return sum(float((o.double() * g.double()).sum()) for o, g in zip(out, grads))
    num = (f(1e-2) - f(-1e-2)) / 2e-2
    assert abs(num - float((d.double() * e.double()).sum())) <= 1e-3 * float(d.norm()) * float(e.norm())


def test_graph_capture_and_replays():
    B, T, Hq, K, Dh = 2, 40, 4, 2, 64
    qkv, grads = _inputs(B, T, Hq, K, Dh, BF)
    sin, cos = _tables(64, Dh)
    at = torch.randint(0, 64, (B, T), device="cuda")
    x = qkv.clone().requires_grad_(True)

    def step():
        out = ops.qkv_norm_rotary(x, Hq, sin, cos, positions=at, num_kv_heads=K)
        return (*out, *torch.autograd.grad(out, [x], grads))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for seed in range(3):
        nx, ng = _inputs(B, T, Hq, K, Dh, BF, seed=seed + 9)
        with torch.no_grad():
            x.copy_(nx), at.copy_(torch.randint(0, 64, (B, T), device="cuda"))
            for a, b in zip(grads, ng):
                a.copy_(b)
        g.replay()
        torch.cuda.synchronize()
        want = _call(nx, Hq, K, sin, cos, ng, positions=at.clone())
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_compiled_matches_eager():
    torch._dynamo.reset()
    B, T, Hq, K, Dh = 2, 10, 4, 2, 64
    qkv, grads = _inputs(B, T, Hq, K, Dh, BF)
    sin, cos = _tables(T, Dh)
    ref = _call(qkv, Hq, K, sin, cos, grads)
    f = torch.compile(lambda t: ops.qkv_norm_rotary(t, Hq, sin, cos, num_kv_heads=K), backend="aot_eager", fullgraph=True)
    x = qkv.clone().requires_grad_(True)
    out = f(x)
    (d,) = torch.autograd.grad(out, [x], grads)
    for a, b in zip((*[o.detach() for o in out], d), ref):
        assert torch.equal(a, b)


def test_refused_calls_and_changed_values():
    """Refusals that need GPU tensors, and writing into the values while their gradient is to come."""
    B, T, Hq, K, Dh = 1, 4, 2, 1, 64
    qkv, grads = _inputs(B, T, Hq, K, Dh, BF)
    sin, cos = _tables(8, Dh)
    bad = [dict(positions=5), dict(positions=-1), dict(positions=True), dict(positions=1.0),
           dict(positions=torch.zeros(T, device="cuda")), dict(positions=torch.zeros(T + 1, device="cuda", dtype=torch.long)),
           dict(positions=torch.zeros((T, B, 1), device="cuda", dtype=torch.long)),
           dict(positions=torch.zeros(T, dtype=torch.long))]
    for kw in bad:
        with pytest.raises(RuntimeError):
            ops.qkv_norm_rotary(qkv, Hq, sin, cos, num_kv_heads=K, **kw)
    with pytest.raises(RuntimeError):
        ops.qkv_norm_rotary(qkv, Hq, sin.cpu(), cos.cpu(), num_kv_heads=K)
    x = qkv.clone().requires_grad_(True)
    _, _, v = ops.qkv_norm_rotary(x, Hq, sin, cos, num_kv_heads=K)
    with pytest.raises(RuntimeError):
        v.add_(1.0)
    # the projection changed in place between forward and backward is noticed
    x = qkv.clone().requires_grad_(True)
    y = x * 1.0
    q, _, _ = ops.qkv_norm_rotary(y, Hq, sin, cos, num_kv_heads=K)
    with torch.no_grad():
        y.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(q, x, grads[0])


def test_general_route_gives_the_same(monkeypatch):
    """The library ops that a traced call uses, run eagerly: the same results as the native call."""
    B, T, Hq, K, Dh = 2, 9, 4, 2, 64
    qkv, grads = _inputs(B, T, Hq, K, Dh, BF)
    sin, cos = _tables(16, Dh)
    at = torch.randint(0, 16, (B, T), device="cuda")
    for kw in (dict(), dict(positions=3), dict(positions=at), dict(positions=at[0], qk_norm=False)):
        ref = _call(qkv, Hq, K, sin, cos, grads, **kw)
        with monkeypatch.context() as m:
            m.setattr(ops, "_native", lambda *names: None)
            got = _call(qkv, Hq, K, sin, cos, grads, **kw)
        assert all(torch.equal(a, b) for a, b in zip(ref, got))


@pytest.mark.parametrize("offset", [0, 1])  # vectors, single values
def test_more_workgroups_than_one_launch_dimension_holds(offset):
    # narrow heads of many tokens: above 2^32 threads; bit for bit as in halves
    B, T, half = 1_060_000, 64, 530_000
    g = torch.Generator(device="cuda").manual_seed(3)
    flat = torch.randn(B * T * 6 + offset, generator=g, device="cuda", dtype=BF)
    qkv = flat[offset:].view(B, T, 6).requires_grad_(True)
    grads = [torch.randn(B, 1, T, 2, generator=g, device="cuda", dtype=BF) for _ in range(3)]
    sin, cos = _tables(T, 2)
    whole = _call(qkv, 1, 1, sin, cos, grads)
    for s in (slice(0, half), slice(half, B)):
        part = _call(qkv[s], 1, 1, sin, cos, [x[s] for x in grads])
        assert all(torch.equal(a[s], b) for a, b in zip(whole, part))
