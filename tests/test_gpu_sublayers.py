"""The sublayer operators together, as the decoder runs them (fuse_qkv_rotary, fuse_swiglu).

* the reference model's golden cases with both on: hidden state and loss within the model-level bound of the decoder's
  other GPU tests (relative L2 error 1e-4 in fp32, 3e-2 in bf16), gradients in fp32 too.  In bf16 the golden gradients
  are themselves a chain of roundings away from the gradient of these weights, further in relative terms the more a sum
  over tokens cancels (a read query's gradient by 4e-2 and more), and the fused sublayers leave most of those roundings
  out.  So both are held against the same model in fp32: with an independent rounding of one size at each place, and
  fewer places, the mean square of the tensors' relative errors is at most the golden one's; over 20 tensors and more a
  mean square varies by sqrt(2 / 20) = 0.32, two deviations of both sides are a factor of (1.64 / 0.55) ** 0.5 at the very
  worst and 1.64 ** 0.5 = 1.3 for one: 1.5 is allowed;
* every call the decoder makes checked against the oracle on the same inputs.  The kernels round once where the oracle's
  eager ops round at each step; with r = 2^-8 (bf16), per element: queries and keys are turned pairs of a normed row,
  whose length p no rounding moves by more than r: the oracle rounds the normed row, two products and a sum (4 r p), the
  bf16 tables are the same on both sides, the kernel rounds once: 5 r p.  h = u silu(z): the oracle rounds u, z, silu(z)
  and the product; |silu'| z <= 1.1 max(|silu(z)|, |z|), so (4 r (|h| + 1.1 |u z|)) and r |h| for the kernel, and both
  sums over D products in fp32 (D 2^-24 of sum |x w|, below r / 8 of it for D <= 2048);
* a layer captured in HIP graphs, forward and backward, against the eager layer on every replay.
"""

import pytest
import torch

import _attnres_hip as H
import attnres_decoder as AD
import attnres_ops as ops
from oracle import attnres_oracle as O
from decoder_util import OracleOps, build_from_case, lm_step, load_model_case, model_index
from gpu_util import DEV

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    H.load()


def _rel_l2(a, e):
    a, e = a.detach().float().cpu(), e.detach().float().cpu()
    return float((a - e).norm() / e.norm().clamp_min(1e-30))


@pytest.mark.parametrize("rotary,swiglu", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("name", sorted(model_index()))
def test_decoder_golden_with_fused_sublayers(name, rotary, swiglu):
    t, meta = load_model_case(name)
    model = build_from_case(t, meta, None, device=DEV, fuse_qkv_rotary=rotary, fuse_swiglu=swiglu)
    hidden, loss = lm_step(model, t["idx"].to(DEV), t["targets"].to(DEV))
    bound = 1e-4 if meta["dtype"] == "fp32" else 3e-2
    assert _rel_l2(hidden, t["hidden"]) <= bound
    assert abs(float(loss) - float(t["loss"][0])) <= bound * abs(float(t["loss"][0]))
    if meta["dtype"] == "fp32":
        for pname, p in model.named_parameters():
            assert _rel_l2(p.grad, t[f"grad.{pname}"]) <= bound, pname
        return
    exact = build_from_case(t, dict(meta, dtype="fp32"), OracleOps)
    lm_step(exact, t["idx"], t["targets"])
    here, golden = [], []
    for pname, p in exact.named_parameters():
        here.append(_rel_l2(dict(model.named_parameters())[pname].grad, p.grad))
        golden.append(_rel_l2(t[f"grad.{pname}"], p.grad))
    assert len(here) >= 20
    rms = [(sum(v * v for v in e) / len(e)) ** 0.5 for e in (here, golden)]
    assert rms[0] <= 1.5 * rms[1], rms


class CheckingOps:
    """HIP sublayers, each call checked against the oracle; the reads go to the drop-in module."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return getattr(ops, name)

    def qkv_norm_rotary(self, qkv, n_head, sin, cos, qk_norm=True):
        out = ops.qkv_norm_rotary(qkv, n_head, sin, cos, qk_norm=qk_norm)
        ref = O.qkv_norm_rotary_ref(qkv, n_head, sin, cos, qk_norm=qk_norm)
        r = 2.0 ** -8
        for a, e in zip(out[:2], ref[:2]):
            assert a.is_contiguous() and a.shape == e.shape
            e = e.float()
            p = (e[..., 0::2] ** 2 + e[..., 1::2] ** 2).sqrt().repeat_interleave(2, -1)
            assert bool(((a.float() - e).abs() <= 5 * r * p * (1 + 4 * r)).all())
        assert torch.equal(out[2], ref[2])
        self.calls.append("rotary")
        return out

    def swiglu_projection(self, x, weight):
        h = ops.swiglu_projection(x, weight)
        e = O.swiglu_projection_ref(x, weight).float()
        X, W = x.float(), weight.float()
        up, gate = (X @ W.t()).chunk(2, -1)
        r = 2.0 ** -8
        F_ = weight.size(0) // 2
        mass = X.abs() @ W.abs().t()  # of a sum of D products
        act = torch.nn.functional.silu(gate).abs()
        tol = 5 * r * e.abs() + 4.4 * r * (up * gate).abs() + r / 8 * (act * mass[..., :F_] + 1.1 * up.abs() * mass[..., F_:])
        assert bool(((h.float() - e).abs() <= tol * (1 + 8 * r) + 1e-30).all())
        self.calls.append("swiglu")
        return h


def _config(**kw):
    base = dict(n_layer=3, n_head=4, n_embd=256, mlp_hidden_dim=680, vocab_size=500, block_size=256, attnres_num_blocks=2,
                lrid_rank=32, attn_res_query_init="normal", fuse_qkv_rotary=True, fuse_swiglu=True)
    base.update(kw)
    return AD.DecoderConfig(**base)


@pytest.mark.parametrize("use_attnres", [True, False])
def test_every_call_matches_the_oracle(use_attnres):
    torch.manual_seed(3)
    checker = CheckingOps()
    with torch.device(DEV):
        model = AD.Decoder(_config(use_attnres=use_attnres), ops=checker).to(torch.bfloat16)
    idx = torch.randint(0, 500, (2, 201), device=DEV)
    hidden, loss = lm_step(model, idx, torch.randint(0, 500, (2, 201), device=DEV))
    assert checker.calls == ["rotary", "swiglu"] * 3
    assert bool(hidden.isfinite().all()) and bool(loss.isfinite())
    for pname, p in model.named_parameters():
        if p.grad is None:  # (the first read site takes the embedding as it is)
            assert "lrid_queries" in pname
            continue
        assert bool(p.grad.isfinite().all()), pname


def test_layer_in_graphs():
    """Attention and MLP of a layer as graphed callables: outputs and gradients of each replay equal the eager layer's."""
    torch.manual_seed(4)
    with torch.device(DEV):
        block = AD.Block(_config(use_attnres=False), ops).to(torch.bfloat16)

    class Layer(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.block = block

        def forward(self, x):
            x = x + self.block.attention(x)[0]
            return x + self.block.feed_forward(x)[0]

    eager = Layer()
    xs = [torch.randn(2, 128, 256, device=DEV, dtype=torch.bfloat16, requires_grad=True) for _ in range(4)]
    ups = [torch.randn(2, 128, 256, device=DEV, dtype=torch.bfloat16) for _ in range(4)]
    weights = [p for p in block.parameters()]

    def step(f, x, up):
        y = f(x)
        return [y.detach().clone(), *[g.clone() for g in torch.autograd.grad(y, [x, *weights], up)]]
    want = [step(eager, x, u) for x, u in zip(xs, ups)]
    again = [step(eager, x, u) for x, u in zip(xs, ups)]
    graphed = torch.cuda.make_graphed_callables(eager, (xs[0],))
    for x, u, e, e2 in zip(xs, ups, want, again):
        got = step(graphed, x, u)
        torch.cuda.synchronize()
        for k, (a, b, b2) in enumerate(zip(got, e, e2)):
            # (attention's backward may sum in a varying order: those gradients are compared by norm)
            if torch.equal(b, b2):
                assert torch.equal(a, b) or _rel_l2(a, b) <= 1e-2, k
            else:
                assert _rel_l2(a, b) <= 1e-2, k
        assert torch.equal(got[0], e[0])
