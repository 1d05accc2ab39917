"""swiglu_projection and the decoder's fused sublayers under autocast.

Under autocast the eager MLP's projection (F.linear) runs in the autocast dtype whatever its operands are, and so does the
operator: its results are those of the operands cast first, bit for bit, on the native, the general and the traced route,
and the gradients come back in the operands' own dtypes.

The decoder with fp32 parameters under bf16 autocast, fused sublayers against eager ones: both are held against the same
model in fp32 without autocast.  The fused one rounds at fewer places, each rounding independent and of one size, so the
mean square of its tensors' relative errors is at most the eager one's; over 20 tensors and more a mean square varies by
sqrt(2 / 20) = 0.32, two deviations of one side are a factor of 1.64 ** 0.5 = 1.3: 1.5 is allowed.
"""

import pytest
import torch
from torch.nn import functional as F

import _attnres_hip as H
import attnres_decoder as AD
import attnres_ops as ops
from decoder_util import lm_step
from gpu_util import DEV

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    H.load()
    H.native()


def _values(n, D, F_, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + n + D + F_)
    rn = lambda *s, std=1.0: torch.randn(s, generator=g, device=DEV) * std  # noqa: E731
    return rn(n, D), rn(2 * F_, D, std=1.5 * D ** -0.5), rn(n, F_)


def _step(f, x, w, dh):
    h = f(x, w)
    return (h, *torch.autograd.grad(h, (x, w), dh.to(h.dtype)))


def _leaves(x, w, xt, wt):
    return x.to(xt).detach().requires_grad_(True), w.to(wt).detach().requires_grad_(True)


@pytest.mark.parametrize("route", ["native", "general", "traced"])
@pytest.mark.parametrize("xt,wt", [(F32, F32), (BF, F32), (F32, BF), (BF, BF), (FP, FP)])
@pytest.mark.parametrize("cast", [BF, FP])
def test_runs_in_the_autocast_dtype(cast, xt, wt, route, monkeypatch):
    f = ops.swiglu_projection
    if route == "general":
        monkeypatch.setattr(ops, "_native", lambda *names: None)
    elif route == "traced":
        torch._dynamo.reset()
        f = torch.compile(ops.swiglu_projection, backend="aot_eager", fullgraph=True)
    for n, D, F_ in ((70, 64, 40), (3, 33, 17)):
        x, w, dh = _values(n, D, F_)
        lx, lw = _leaves(x, w, xt, wt)
        with torch.autocast(DEV, cast):
            got = _step(f, lx, lw, dh)
            assert F.linear(lx, lw).dtype == got[0].dtype == cast
        cx, cw = _leaves(lx.detach(), lw.detach(), cast, cast)
        want = _step(ops.swiglu_projection, cx, cw, dh)
        assert torch.equal(got[0], want[0])
        for a, e, t in zip(got[1:], want[1:], (xt, wt)):
            assert a.dtype == t and torch.equal(a, e.to(t))


def test_what_autocast_leaves_alone():
    x, w, dh = _values(20, 64, 40)
    want = ops.swiglu_projection(x, w)
    with torch.autocast(DEV, BF):
        with torch.autocast(DEV, enabled=False):
            got = ops.swiglu_projection(x, w)
        assert got.dtype == F32 and torch.equal(got, want)
        # fp64 is never cast by autocast: the weight is taken in the input's dtype, the input is refused
        h = ops.swiglu_projection(x.to(BF), w.double())
        assert torch.equal(h, ops.swiglu_projection(x.to(BF), w.double().to(BF)))
        with pytest.raises(RuntimeError, match="dtype"):
            ops.swiglu_projection(x.double(), w)
    with torch.autocast("cpu", BF):  # another device's
        assert torch.equal(ops.swiglu_projection(x, w), want)


def test_a_weight_used_twice_and_first_without_gradients():
    """The cast weight that autocast keeps for its context must not lose the weight's gradient."""
    x, w, dh = _values(40, 64, 40)
    lw = w.clone().requires_grad_(True)
    with torch.autocast(DEV, BF):
        with torch.no_grad():
            first = ops.swiglu_projection(x, lw)
        a = ops.swiglu_projection(x, lw)
        b = ops.swiglu_projection(x, lw)
    assert torch.equal(first, a.detach()) and torch.equal(a, b)
    (g,) = torch.autograd.grad((a, b), lw, (dh.to(BF), dh.to(BF)))
    cw = w.to(BF).requires_grad_(True)
    (e,) = torch.autograd.grad(ops.swiglu_projection(x.to(BF), cw), cw, dh.to(BF))
    assert g.dtype == F32 and torch.equal(g, 2 * e.float())


class _Noting:
    """The drop-in module's functions, noting the dtypes that the sublayers' operators take and give."""

    def __init__(self):
        self.seen = []

    def __getattr__(self, name):
        return getattr(ops, name)

    def qkv_norm_rotary(self, qkv, *args, **kw):
        out = ops.qkv_norm_rotary(qkv, *args, **kw)
        self.seen.append(("rotary", qkv.dtype, *(t.dtype for t in out)))
        return out

    def swiglu_projection(self, x, weight):
        h = ops.swiglu_projection(x, weight)
        self.seen.append(("swiglu", weight.dtype, h.dtype))
        return h


def _rel_l2(a, e):
    a, e = a.detach().float().cpu(), e.detach().float().cpu()
    return float((a - e).norm() / e.norm().clamp_min(1e-30))


def test_decoder_with_fp32_parameters_under_autocast():
    base = dict(n_layer=4, n_head=4, n_embd=256, mlp_hidden_dim=680, vocab_size=500, block_size=256, use_attnres=False)
    noting = _Noting()
    torch.manual_seed(3)
    with torch.device(DEV):
        fused = AD.Decoder(AD.DecoderConfig(**base, fuse_qkv_rotary=True, fuse_swiglu=True), ops=noting)
        eager, exact = AD.Decoder(AD.DecoderConfig(**base)), AD.Decoder(AD.DecoderConfig(**base))
    eager.load_state_dict(fused.state_dict())
    exact.load_state_dict(fused.state_dict())
    idx, targets = (torch.randint(0, 500, (2, 201), device=DEV) for _ in range(2))
    want = lm_step(exact, idx, targets)
    errors = []
    for model in (fused, eager):
        with torch.autocast(DEV, BF):
            hidden, loss = lm_step(model, idx, targets)
        grads = {name: p.grad for name, p in model.named_parameters()}
        assert all(g.dtype == F32 for g in grads.values())
        errors.append([_rel_l2(hidden, want[0])] + [_rel_l2(grads[name], p.grad) for name, p in exact.named_parameters()])
    assert noting.seen == [("rotary", BF, BF, BF, BF), ("swiglu", F32, BF)] * 4
    assert len(errors[0]) >= 18
    rms = [(sum(v * v for v in e) / len(e)) ** 0.5 for e in errors]
    assert 0.0 < rms[0] <= 1.5 * rms[1], rms
