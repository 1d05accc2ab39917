"""What swiglu_projection keeps of u and z for its backward: 12 (bf16) and 16 (fp16) significant bits, the 16 highest of
the fp32 value in one plane and the other 4 or 8 in another.

* exactly: inputs whose u, or z, needs those bits and no more, each element of its own, and whose results are exact sums
  rounded once.  The projections' gradient is rounded to the dtype from all of the kept bits, so that dx and dweight,
  compared bit for bit, change with a low bit that is dropped, swapped or read from another element's place;
* values: random inputs against 64 bits.  As in test_gpu_swiglu.py (u = 2^-24, r = eps / 2), but with what is kept counted
  as what it is: eu = k |u| + D u U and ez = k |z| + D u Z off, with k = 2^-12 (bf16), 2^-16 (fp16), 0 (fp32) the half
  step of the kept bits.
"""

import pytest
import torch

import _attnres_hip as H
import attnres_ops as ops

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
KEPT = {BF: 2.0 ** -12, FP: 2.0 ** -16, F32: 0.0}


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


def _case(which, n, D, F, dtype, seed=0):
    """x[:, 0] = 1, x[:, 1:] = -1 or 1 steps of 2^-6 (bf16) or 2^-10 (fp16).  The projection `which` ("u" or "z") has
    whole weights 19 .. 61 in column 0 and up to twelve whole ones a row elsewhere: its values are multiples of the step
    between 17 and 63, of 11 and 12 or 15 and 16 significant bits.  From 17 on silu(z) = z and silu'(z) = 1 to the last
    bit (exp(-17) < 2^-24).  The other projection: z = 64 in every element, or u = 1, -1 or 0.

    Exact sums: rounded, such a value is a multiple of 2^-3 (bf16) or 2^-6 (fp16) below 64, so with |dh| <= 1 the terms
    of dx are multiples of 1 (u's case: dz times 64 or 0, du = 64 dh times whole weights) or 2^-6 (z's: du times 1, -1 or
    0, dz whole), at most 64 * 64 + 64 * 61 or 64 + 61 of them a hidden value; those of dweight multiples of 2^-16
    at most (2^-6 times a step of x), and one column's all of the same size.  Below 2^24 steps for F <= 2000, n <= 4000."""
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * n + 10 * D + F)

    def ints(shape, lo, hi):
        return torch.randint(lo, hi + 1, shape, generator=g, device="cuda").double()

    step, most = (2.0 ** -6, 7) if dtype == BF else (2.0 ** -10, 63)
    x = (2 * ints((n, D), 0, 1) - 1) * step
    x[:, 0] = 1
    w = torch.zeros((2 * F, D), device="cuda", dtype=torch.float64)
    few = torch.rand((F, D), generator=g, device="cuda").argsort(1) < 12
    full = ints((F, D), -most, most) * few
    full[:, 0] = ints((F,), 19, 61)
    if which == "u":
        w[:F], w[F:, 0] = full, 64
    else:
        w[F:], w[:F, 0] = full, ints((F,), -1, 1)
    dh = ints((n, F), -1, 1)
    u, z = x @ w[:F].t(), x @ w[F:].t()
    mine = u if which == "u" else z
    assert 17 <= float(mine.min()) and float(mine.max()) <= 63 and torch.equal(mine / step, (mine / step).round())
    # what the high plane alone would give is another value for many elements
    high = mine.float().view(torch.int32).bitwise_and(-65536).view(F32)
    assert float((high.to(dtype) != mine.to(dtype)).float().mean()) > 0.2
    du, dz = (dh * z).to(dtype).double(), (dh * u).to(dtype).double()
    d = torch.cat([du, dz], dim=1)
    return x, w, dh, u * z, d @ w, d.t() @ x


# up to 64 tokens, then every tile of the forward, whole and split over k: 64 x 128, 128 x 128, 256 x 256
SHAPES = [(1, 40, 32), (5, 40, 33), (17, 64, 65), (64, 200, 72), (106, 98, 302), (93, 2106, 70), (1864, 49, 1820),
          (2913, 2966, 82), (3511, 131, 1941), (3671, 3239, 536)]


@pytest.mark.parametrize("which", ["u", "z"])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("n,D,F", SHAPES)
def test_every_kept_bit(n, D, F, dtype, which):
    x, w, dh, h, dx, dw = _case(which, n, D, F, dtype)
    assert torch.equal(x.to(dtype).double(), x) and torch.equal(w.to(dtype).double(), w)
    got = _run(x.to(dtype), w.to(dtype), dh.to(dtype))
    for name, a, e in zip(("h", "dx", "dw"), got, (h, dx, dw)):
        e = e.float().to(dtype)
        assert torch.equal(a, e), (name, int((a != e).sum()), a.numel())


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("n,D,F", [(1, 64, 32), (50, 200, 136), (333, 256, 300), (1500, 500, 363), (93, 2106, 70)])
def test_values(n, D, F, dtype):
    g = torch.Generator(device="cuda").manual_seed(7 + n + D + F)
    rn = lambda *s, std=1.0: (torch.randn(s, generator=g, device="cuda") * std).to(dtype)  # noqa: E731
    x, w, dh = rn(n, D), rn(2 * F, D, std=1.5 * D ** -0.5), rn(n, F)
    _, gx, gw = _run(x, w, dh)
    r, k = torch.finfo(dtype).eps / 2, KEPT[dtype]
    X, W, G = x.double(), w.double(), dh.double()
    u, z = X @ W[:F].t(), X @ W[F:].t()
    s = torch.sigmoid(z)
    silu, dsilu = z * s, s * (1 + z * (1 - s))
    du, dz = G * silu, G * u * dsilu
    au, az = X.abs() @ W[:F].abs().t(), X.abs() @ W[F:].abs().t()
    act = 2.0 ** -20 * (1 + z.abs() / 8)
    eu, ez = k * u.abs() + D * U * au, k * z.abs() + D * U * az
    tiny = float(torch.finfo(dtype).tiny)  # (below it a rounding is half a step of the smallest values)
    tu = G.abs() * 1.1 * ez + (r + act) * du.abs() + r * tiny
    tz = G.abs() * (1.1 * eu + 0.5 * u.abs() * ez) + r * dz.abs() + 4 * act * (G * u).abs() * 1.1 + r * tiny
    d, t = torch.cat([du, dz], 1), torch.cat([tu, tz], 1)
    dx, dw = d @ W, d.t() @ X
    tx = t @ W.abs() + 2 * F * U * (d.abs() @ W.abs()) + r * dx.abs()
    tw = t.t() @ X.abs() + n * U * (d.abs().t() @ X.abs()) + r * dw.abs()
    for name, a, e, tol in (("dx", gx, dx, tx), ("dw", gw, dw, tw)):
        off = (a.double() - e).abs()
        assert not bool((off > 1.05 * tol + r * tiny).any()), (name, float((off / (tol + r * tiny)).max()))
