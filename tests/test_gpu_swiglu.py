"""The gated feed-forward projections (swiglu_projection), forward and backward.

* every product counted once: integer inputs whose gate saturates (z = 64 in every row, silu(64) = 64 and silu'(64) = 1
  to the last bit), so that u, h and the projections' gradient are exact in every dtype and the results are the exact
  sums rounded once -- compared bit for bit over token counts, widths, row strides and dtypes around every tile, chunk
  and k step;
* values: random inputs against 64 bits, element by element.

Tolerances (u = 2^-24, r = eps / 2 of the dtype: a rounding's largest relative error).  A sum of K products in fp32 in
any order is within K u sum |x w| of the exact one.  With U = sum |x Wu|, Z = sum |x Wg|, |silu'| <= 1.1, |silu''| <= 0.5
and a silu computed to 2^-20 (1 + |z| / 8) (exp2 of a rounded product, a reciprocal and two products):
  |dh| <= r |h| + (D + 4) u (1.1 |u| Z + |silu(z)| U) + 2^-20 (1 + |z| / 8) |h|
The backward reads u and z as the forward summed and rounded them, eu = r |u| + D u U and ez = r |z| + D u Z off (in fp32,
where r = u, and where a sum cancels, the second term is the larger one), and rounds [du dz]:
  |ddu| <= |g| 1.1 ez + (r + 2^-20 (1 + |z| / 8)) |du|
  |ddz| <= |g| (1.1 eu + 0.5 |u| ez) + (r + 2^-18 (1 + |z| / 8)) |g u| 1.1
and the products add K u sum |d| |w| and one rounding.  Second-order terms are counted by a factor of 1.05 on the whole.
"""

import pytest
import torch

import _attnres_hip as H
import attnres_ops as ops

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    H.load()
    H.native()


def _ints(g, shape, lo, hi):
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda").double()


def _exact_case(n, D, F, dtype, seed=0):
    """x[:, 0] = 1 and gate weights [64, 0, ...]: z = 64.  Other values -1, 0, 1, mostly zero, so that |u| stays small."""
    g = torch.Generator(device="cuda").manual_seed(1000 * n + 10 * D + F + seed)
    keep = min(1.0, 24.0 / D)
    x = _ints(g, (n, D), -1, 1)
    x[:, 0] = 1
    w = torch.zeros((2 * F, D), device="cuda", dtype=torch.float64)
    w[:F] = _ints(g, (F, D), -1, 1) * (torch.rand((F, D), generator=g, device="cuda") < keep)
    w[F:, 0] = 64
    dh = _ints(g, (n, F), -2, 2)
    u = x @ w[:F].t()
    assert float(u.abs().max()) <= 60  # (2 u and 64 u are exact in 8 bits)
    h = u * 64
    d = torch.cat([dh * 64, dh * u], dim=1)
    return x, w, dh, h, d @ w, d.t() @ x


def _run(x, w, dh, want=(True, True)):
    x, w = x.detach().requires_grad_(want[0]), w.detach().requires_grad_(want[1])
    h = ops.swiglu_projection(x, w)
    leaves = [t for t, k in zip((x, w), want) if k]
    grads = list(torch.autograd.grad(h, leaves, dh))
    return h.detach(), grads.pop(0) if want[0] else None, grads.pop(0) if want[1] else None


def _check_exact(n, D, F, dtype, lay=lambda t: t, lay_w=lambda t: t, lay_g=lambda t: t):
    x, w, dh, h, dx, dw = _exact_case(n, D, F, dtype)
    a = _run(lay(x.to(dtype)), lay_w(w.to(dtype)), lay_g(dh.to(dtype)))
    for name, got, e in zip(("h", "dx", "dw"), a, (h, dx, dw)):
        e = e.float().to(dtype)  # (sums below 2^24: exact in fp32, rounded once)
        assert torch.equal(got, e), (name, n, D, F, dtype, int((got != e).sum()), got.numel())


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 33, 64, 65, 129, 300])
def test_token_counts(n, dtype):
    _check_exact(n, 96, 72, dtype)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("D", [1, 2, 7, 8, 24, 31, 32, 33, 40, 130, 256, 264, 515])
def test_widths(D, dtype):
    _check_exact(37, D, 40, dtype)


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("F", [1, 3, 8, 16, 31, 32, 33, 64, 65, 127, 128, 200, 257, 520])
def test_hidden_widths(F, dtype):
    _check_exact(45, 64, F, dtype)


@pytest.mark.parametrize("n,D,F", [(2048, 512, 1024), (1031, 776, 520), (4099, 256, 264), (515, 1030, 1001),
                                   (8192, 64, 32), (40, 1024, 4096), (1, 768, 2048), (9, 2048, 250), (5000, 40, 2000)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_large(n, D, F, dtype):
    _check_exact(n, D, F, dtype)


# together these take every tile of every product, whole and split over k, in 16 bits and in fp32
TILES = [(65, 36, 49), (1758, 73, 2148), (1429, 1459, 814), (3568, 162, 1978), (6469, 2187, 485), (1363, 1750, 1904),
         (4788, 1649, 46), (3729, 1840, 1258), (2202, 1913, 2240)]


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("n,D,F", TILES)
def test_every_tile_and_split(n, D, F, dtype):
    _check_exact(n, D, F, dtype)


def _strided(t, pad, offset=0):
    big = torch.full((t.size(0), t.size(1) + pad), float("nan"), device=t.device, dtype=t.dtype)
    big[:, offset:offset + t.size(1)] = t
    return big[:, offset:offset + t.size(1)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("pad,offset", [(8, 0), (8, 8), (3, 0), (5, 1)])
def test_row_strides_and_alignment(pad, offset, dtype):
    _check_exact(70, 64, 48, dtype, *[lambda t: _strided(t, pad, offset)] * 3)


def test_transposed_and_expanded_operands():
    _check_exact(70, 64, 48, BF, lambda t: t.t().contiguous().t(), lambda t: t.t().contiguous().t(),
                 lambda t: t.t().contiguous().t())
    x, w = torch.ones((1, 32), device="cuda", dtype=BF).expand(5, 32), torch.ones((64, 32), device="cuda", dtype=BF)
    assert torch.equal(ops.swiglu_projection(x, w), ops.swiglu_projection(x.contiguous(), w))
    w1 = torch.full((1, 32), 0.125, device="cuda", dtype=BF).expand(6, 32)
    assert torch.equal(ops.swiglu_projection(x, w1), ops.swiglu_projection(x, w1.contiguous()))


def _values(n, D, F, dtype, seed=0, scale=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed + n + D + F)
    rn = lambda *s, std=1.0: (torch.randn(s, generator=g, device="cuda") * std).to(dtype)  # noqa: E731
    return rn(n, D), rn(2 * F, D, std=scale * D ** -0.5), rn(n, F)


def _check_values(x, w, dh):
    n, D = x.shape
    F = w.size(0) // 2
    r = torch.finfo(x.dtype).eps / 2
    a = _run(x, w, dh)
    X, W, G = x.double(), w.double(), dh.double()
    u, z = X @ W[:F].t(), X @ W[F:].t()
    s = torch.sigmoid(z)
    silu, dsilu = z * s, s * (1 + z * (1 - s))
    h, du, dz = u * silu, G * silu, G * u * dsilu
    au, az = X.abs() @ W[:F].abs().t(), X.abs() @ W[F:].abs().t()
    act = 2.0 ** -20 * (1 + z.abs() / 8)
    th = r * h.abs() + (D + 4) * U * (1.1 * u.abs() * az + silu.abs() * au) + act * h.abs()
    eu, ez = r * u.abs() + D * U * au, r * z.abs() + D * U * az
    tu = G.abs() * 1.1 * ez + (r + act) * du.abs()
    tz = G.abs() * (1.1 * eu + 0.5 * u.abs() * ez) + (r + 4 * act) * (G * u).abs() * 1.1
    d, t = torch.cat([du, dz], 1), torch.cat([tu, tz], 1)
    dx, dw = d @ W, d.t() @ X
    tx = t @ W.abs() + 2 * F * U * (d.abs() @ W.abs()) + r * dx.abs()
    tw = t.t() @ X.abs() + n * U * (d.abs().t() @ X.abs()) + r * dw.abs()
    tiny = float(torch.finfo(x.dtype).tiny)
    for name, got, e, tol in zip(("h", "dx", "dw"), a, (h, dx, dw), (th, tx, tw)):
        off = (got.double() - e).abs()
        bad = off > 1.05 * tol + tiny
        assert not bool(bad.any()), (name, float((off / (tol + tiny)).max()))


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("n,D,F", [(1, 64, 32), (50, 200, 136), (333, 256, 300), (1500, 500, 363)])
def test_values(n, D, F, dtype):
    _check_values(*_values(n, D, F, dtype))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_wide_range_of_gates(dtype):
    x, w, dh = _values(64, 128, 96, dtype, scale=20.0)  # |z| to about 80
    _check_values(x, w, dh)


def test_difference_quotients():
    """The gradient against central differences of the forward, in fp32: the step's third-order term (1e-2^2 / 6 of the
    third derivative) and the forward's rounding over the step both stay below 1e-3 of the gradients' size."""
    x, w, dh = _values(6, 40, 24, F32, seed=3)
    _, dx, dw = _run(x, w, dh)
    for t, g in ((x, dx), (w, dw)):
        e = torch.randn(t.shape, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
        step = 1e-2

        def f(s):
            a, b = (x + s * e, w) if t is x else (x, w + s * e * 0.1)
            return float((ops.swiglu_projection(a, b).double() * dh.double()).sum())
        scale = 1.0 if t is x else 0.1
        num = (f(step) - f(-step)) / (2 * step)
        assert abs(num - scale * float((g.double() * e.double()).sum())) <= 2e-3 * scale * float(g.norm()) * float(e.norm()) / 10


def test_infinities_and_nan_stay_in_their_rows():
    x, w, _ = _values(40, 64, 48, BF)
    clean = ops.swiglu_projection(x, w)
    x2 = x.clone()
    x2[3] = float("nan")
    x2[17, 5] = float("inf")
    h = ops.swiglu_projection(x2, w)
    rows = [i for i in range(40) if i not in (3, 17)]
    assert torch.equal(h[rows], clean[rows])
    assert bool(h[3].isnan().all()) and not bool(h[17].isfinite().any())
    wz = w.clone()
    wz[10] = float("inf")  # an up row: that column alone
    h = ops.swiglu_projection(x, wz)
    cols = [i for i in range(48) if i != 10]
    assert torch.equal(h[:, cols], clean[:, cols]) and not bool(h[:, 10].isfinite().any())


def test_ragged_k_ends_do_not_mix_operands():
    """A last hidden row or token that is infinite stays out of everything it has no part in, also where the last k step
    is not full (hidden 33: one row in its step)."""
    x, w, dh = _values(33, 64, 33, BF)
    ref = _run(x, w, dh)
    dh2 = dh.clone()
    dh2[32] = float("nan")
    got = _run(x, w, dh2)
    assert torch.equal(got[1][:32], ref[1][:32]) and bool(got[1][32].isnan().all())


@pytest.mark.parametrize("want", [(True, False), (False, True)])
def test_one_gradient_alone(want):
    x, w, dh = _values(130, 96, 80, BF)
    both, one = _run(x, w, dh), _run(x, w, dh, want)
    for a, b, k in zip(both[1:], one[1:], want):
        assert (b is None) if not k else torch.equal(a, b)


def test_shapes_empty_and_no_grad():
    x, w, dh = _values(24, 32, 16, BF)
    ref = ops.swiglu_projection(x, w)
    assert torch.equal(ops.swiglu_projection(x.view(2, 3, 4, 32), w), ref.view(2, 3, 4, 16))
    assert torch.equal(ops.swiglu_projection(x[5], w), ops.swiglu_projection(x[5:6], w)[0])
    xe = torch.empty((2, 0, 32), device="cuda", dtype=BF, requires_grad=True)
    wl = w.clone().requires_grad_(True)
    h = ops.swiglu_projection(xe, wl)
    assert h.shape == (2, 0, 16)
    h.sum().backward()
    assert xe.grad.shape == xe.shape and float(wl.grad.abs().max()) == 0.0
    with torch.no_grad():
        assert torch.equal(ops.swiglu_projection(x.requires_grad_(True), w), ref)
    # a weight of another dtype is taken in x's, its gradient comes back in its own
    w32 = w.float().requires_grad_(True)
    h = ops.swiglu_projection(x.detach(), w32)
    assert torch.equal(h.detach(), ref)
    (g,) = torch.autograd.grad(h, w32, dh)
    assert g.dtype == F32 and torch.equal(g, _run(x.detach(), w, dh)[2].float())


def test_repeats_bit_for_bit_and_expanded_gradient():
    x, w, dh = _values(700, 160, 200, BF)
    a, b = _run(x, w, dh), _run(x, w, dh)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    one = torch.ones((), device="cuda", dtype=BF).expand(700, 200)
    a, b = _run(x, w, one), _run(x, w, one.contiguous())
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_second_order_is_refused():
    x, w, dh = _values(8, 32, 16, F32)
    x.requires_grad_(True)
    (g,) = torch.autograd.grad(ops.swiglu_projection(x, w), x, dh.requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError, match="twice|once_differentiable"):
        g.sum().backward()


def test_another_stream_and_saved_tensor_hooks():
    x, w, dh = _values(300, 96, 80, BF)
    ref = _run(x, w, dh)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _run(x, w, dh)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(ref, got))

    def other_layout(t):  # the same values, another memory layout (and alignment)
        if t.dim() > 1:
            return t.transpose(-1, -2).contiguous().transpose(-1, -2)
        return torch.cat([t.new_zeros(1), t])[1:]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, other_layout):
        got = _run(x, w, dh)
    assert all(torch.equal(p, q) for p, q in zip(ref, got))


def test_graph_capture_and_replays():
    """Forward and backward captured once, replayed on new inputs with eager work between; every replay equals eager."""
    n, D, F = 300, 96, 80
    x, w, dh = (t.clone() for t in _values(n, D, F, BF))
    x.requires_grad_(True), w.requires_grad_(True)

    def step():
        h = ops.swiglu_projection(x, w)
        return (h, *torch.autograd.grad(h, (x, w), dh))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for seed in range(3):
        nx, nw, nd = _values(n, D, F, BF, seed=50 + seed)
        with torch.no_grad():
            x.copy_(nx), w.copy_(nw), dh.copy_(nd)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, _run(nx, nw, nd)))


def test_compiled_matches_eager():
    torch._dynamo.reset()
    x, w, dh = _values(70, 64, 40, BF)
    ref = _run(x, w, dh)
    f = torch.compile(ops.swiglu_projection, backend="aot_eager", fullgraph=True)
    x.requires_grad_(True), w.requires_grad_(True)
    h = f(x, w)
    got = (h.detach(), *torch.autograd.grad(h, (x, w), dh))
    assert all(torch.equal(a, b) for a, b in zip(ref, got))


def test_general_route_gives_the_same(monkeypatch):
    """The library ops that a traced call uses, run eagerly: the same results as the native call."""
    for n, D, F in ((70, 64, 40), (5, 33, 17)):
        x, w, dh = _values(n, D, F, BF)
        ref = _run(x, w, dh)
        with monkeypatch.context() as m:
            m.setattr(ops, "_native", lambda *names: None)
            got = _run(x, w, dh)
            with torch.no_grad():
                again = ops.swiglu_projection(x, w)
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)):
                moved = _run(x, w, dh)
        assert all(torch.equal(a, b) for a, b in zip(ref, got)) and torch.equal(again, ref[0])
        assert all(torch.equal(a, b) for a, b in zip(ref, moved))


def test_two_calls_at_once_on_two_streams():
    """Two calls with workspaces of their own (copied operands, split sums) on two streams, several times over."""
    args = [_values(300, 1000, 130, BF, seed=s) for s in (1, 2)] + [_values(90, 130, 77, F32, seed=s) for s in (3, 4)]
    want = [_run(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for a, s in zip(args, streams):
            with torch.cuda.stream(s):
                got.append(_run(*a))
        torch.cuda.synchronize()
        for g, e in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(g, e))


def test_two_captured_graphs_interleaved():
    """Two graphs of calls with workspaces, replayed in turn and together with eager work, each from its own pool."""
    sets = [[t.clone() for t in _values(200, 1000, 130, BF, seed=s)] for s in (5, 6)]
    want = [_run(*a) for a in sets]
    graphs, outs = [], []
    for x, w, dh in sets:
        x.requires_grad_(True), w.requires_grad_(True)

        def step():
            h = ops.swiglu_projection(x, w)
            return (h, *torch.autograd.grad(h, (x, w), dh))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for k in (0, 1, 1, 0, 1, 0):
        for t in outs[k]:
            t.detach().zero_()
        graphs[k].replay()
        eager = _run(*[t.detach() for t in sets[1 - k]])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[k], want[k]))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[1 - k]))
