"""The products' kernels that no shape of test_gpu_swiglu.py takes: the 16-bit forward's 256 x 256 and 128 x 128 tiles
split over k, and the fp32 weight gradient's 128 x 256 tile unsplit.  Exact whole sums, compared bit for bit."""

import pytest
import torch

import _attnres_hip as H
import attnres_ops as ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    H.load()
    H.native()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,D,F", [(1447, 7540, 1928), (5567, 5432, 157), (662, 6650, 1195), (3671, 3239, 536),
                                   (2913, 2966, 82)])
def test_split_forwards_and_whole_weight_gradients(n, D, F, dtype):
    """z = 64 (silu(64) = 64, silu'(64) = 1); u a sum of about 20 terms -1 or 1, below 61: u, 64 u and the projections'
    gradient are exact in every dtype, the sums below 2^24 steps of 1."""
    g = torch.Generator(device="cuda").manual_seed(n + D + F)
    ints = lambda s, m: torch.randint(-m, m + 1, s, generator=g, device="cuda").double()  # noqa: E731
    x = ints((n, D), 1)
    x[:, 0] = 1
    w = torch.zeros((2 * F, D), device="cuda", dtype=torch.float64)
    w[:F] = ints((F, D), 1) * (torch.rand((F, D), generator=g, device="cuda") < 24 / D)
    w[F:, 0] = 64
    dh = ints((n, F), 2)
    u = x @ w[:F].t()
    assert float(u.abs().max()) <= 60
    d = torch.cat([dh * 64, dh * u], dim=1)
    lx, lw = x.to(dtype).requires_grad_(True), w.to(dtype).requires_grad_(True)
    h = ops.swiglu_projection(lx, lw)
    dx, dw = torch.autograd.grad(h, (lx, lw), dh.to(dtype))
    for name, a, e in (("h", h.detach(), u * 64), ("dx", dx, d @ w), ("dw", dw, d.t() @ x)):
        e = e.float().to(dtype)
        assert torch.equal(a, e), (name, int((a != e).sum()), a.numel())
