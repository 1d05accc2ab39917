"""Far memory: row strides at the border of the products' 32-bit load offsets, weights and intermediates whose bytes pass
2^32, and the rotary backward on rows beyond 2^31 elements.  Every result is bit for bit that of the dense call (the same
sums in the same order), or the exact one."""

import pytest
import torch

import _attnres_hip as H
import attnres_ops as ops

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    H.load()
    H.native()


def _run(x, w, dh):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    h = ops.swiglu_projection(x, w)
    return (h.detach(), *torch.autograd.grad(h, (x, w), dh))


def _values(n, D, F, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + n + D + F)
    rn = lambda *s, std=1.0: (torch.randn(s, generator=g, device="cuda") * std).to(BF)  # noqa: E731
    return rn(n, D), rn(2 * F, D, std=1.5 * D ** -0.5), rn(n, F)


def _far(t, stride):
    """t with rows `stride` elements apart; what lies between is not initialised"""
    big = torch.empty(((t.size(0) - 1) * stride + t.size(1),), device="cuda", dtype=t.dtype)
    view = big.as_strided(t.shape, (stride, 1))
    view.copy_(t)
    return view


D0 = 64
FAR = 2 ** 32 // (256 * 2) - D0  # rows of a tile up to 256: the last stride that 32-bit offsets reach


@pytest.mark.parametrize("stride", [FAR - 8, FAR, FAR + 8, FAR + 3])
def test_strides_around_the_direct_loads_reach(stride):
    """65 rows of x (tiled products; rows of the forward's tile lie up to 65 strides apart), 1.1 GB."""
    x, w, dh = _values(65, D0, 48)
    want = _run(x, w, dh)
    got = _run(_far(x, stride), w, dh)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    few = [t[:40] for t in (x, dh)]  # up to 64 tokens: the forward's own kernel
    want = _run(few[0], w, few[1])
    got = _run(_far(few[0], stride), w, few[1])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("F,stride", [(128, FAR + D0 - 8), (128, FAR - 8), (129, FAR - 8), (132, FAR - 8), (20, FAR + 8)])
def test_weights_that_span_4_gib(F, stride):
    """2 F rows of the weight just inside 2^32 bytes, beyond them, and at a stride that no tile reaches."""
    x, w, dh = _values(70, D0, F)
    want = _run(x, w, dh)
    got = _run(x, _far(w, stride), dh)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_gradients_with_far_rows():
    x, w, dh = _values(65, D0, 48)
    want = _run(x, w, dh)
    got = _run(x, w, _far(dh, 2 ** 25 + 8))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_intermediates_above_4_gib():
    """[du dz], and what is kept of u and z, end beyond 2^32 bytes: exact whole sums, every token and hidden column."""
    n, D, F = 131101, 24, 8200
    g = torch.Generator(device="cuda").manual_seed(11)
    x = torch.randint(-1, 2, (n, D), generator=g, device="cuda").to(BF)
    x[:, 0] = 1
    w = torch.zeros((2 * F, D), device="cuda", dtype=BF)
    w[:F] = torch.randint(-1, 2, (F, D), generator=g, device="cuda").to(BF)
    w[F:, 0] = 64  # silu(64) = 64, silu'(64) = 1
    dh = torch.randint(-1, 2, (n, F), generator=g, device="cuda").to(BF)
    h, dx, dw = _run(x, w, dh)
    # |u| <= 24: u, 64 u and 64 dh are exact in bf16, and every sum below 2^24 steps of 1 (dw: 64 n < 2^24; dx: |64 dh w +
    # 64 dh u| F < 2^24 steps of 64)
    W = w[:F].double()
    ex = torch.empty((n, D), device="cuda")
    eu, eg = (torch.zeros((F, D), device="cuda", dtype=torch.float64) for _ in range(2))
    for s in range(0, n, 16384):
        X, G = x[s:s + 16384].double(), dh[s:s + 16384].double()
        u = X @ W.t()
        assert torch.equal(h[s:s + 16384].double(), (64 * u).to(BF).double())
        du, dz = 64 * G, G * u
        e = du @ W
        e[:, 0] += 64 * dz.sum(1)
        ex[s:s + 16384] = e.float()
        eu += du.t() @ X
        eg += dz.t() @ X
    assert torch.equal(dx, ex.to(BF))
    assert torch.equal(dw[:F], eu.float().to(BF)) and torch.equal(dw[F:], eg.float().to(BF))


@pytest.mark.parametrize("offset", [0, 1])  # vectors, single values
def test_rotary_rows_beyond_2_to_31_elements(offset):
    """Projection and all three gradients, forward and backward."""
    B, T, Hq, K, Dh = 1, 3, 2, 1, 64
    C, stride = (Hq + 2 * K) * Dh, 2 ** 30 + 64
    g = torch.Generator(device="cuda").manual_seed(2)
    rn = lambda *s: torch.randn(s, generator=g, device="cuda").to(BF)  # noqa: E731
    small, grads = rn(B, T, C), [rn(B, h, T, Dh) for h in (Hq, K, K)]
    a = torch.outer(torch.arange(8, device="cuda"), torch.rand(Dh // 2, generator=g, device="cuda"))
    sin, cos = a.sin(), a.cos()

    def run(qkv, up):
        qkv = qkv.detach().requires_grad_(True)
        out = ops.qkv_norm_rotary(qkv, Hq, sin, cos, num_kv_heads=K)
        return (*(t.detach() for t in out), *torch.autograd.grad(out, [qkv], up))

    def apart(t, shape, strides):
        big = torch.empty((sum((n - 1) * s for n, s in zip(shape, strides)) + 1 + offset,), device="cuda", dtype=BF)
        view = big[offset:].as_strided(shape, strides)
        view.copy_(t)
        return view
    far = apart(small, small.shape, (0, stride, 1))
    if offset:  # (the general kernel adds in another order: the same one on both sides)
        small = apart(small, small.shape, (0, C, 1))
    want = run(small, grads)
    got = run(far, [apart(t, t.shape, (0, Dh, stride, 1)) for t in grads])
    assert all(torch.equal(p, q) for p, q in zip(got, want))
