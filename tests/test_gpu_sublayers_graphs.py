"""The MLP, and a layer, captured in HIP graphs: bit for bit the eager gradients where their sums have a fixed order.

The MLP's own gradients (its input's, fc1's and fc2's) are sums in a fixed order on both sides; attention's backward may
add in a varying one, so what passes through it (the layer's input, c_attn) is compared by norm, in
test_gpu_sublayers.py.  A replay that reads a stale or shared workspace shows here whatever its size."""

import pytest
import torch

import _attnres_hip as H
import attnres_decoder as AD
import attnres_ops as ops
from gpu_util import DEV

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")
    H.load()


class _Layer(torch.nn.Module):
    def __init__(self, block, attention):
        super().__init__()
        self.block, self.attention = block, attention

    def forward(self, x):
        if self.attention:
            x = x + self.block.attention(x)[0]
        return x + self.block.feed_forward(x)[0]


@pytest.mark.parametrize("attention", [False, True])
def test_replays_equal_the_eager_layer(attention):
    torch.manual_seed(4)
    config = AD.DecoderConfig(n_layer=3, n_head=4, n_embd=256, mlp_hidden_dim=680, vocab_size=500, block_size=256,
                              use_attnres=False, fuse_qkv_rotary=True, fuse_swiglu=True)
    with torch.device(DEV):
        block = AD.Block(config, ops).to(BF)
    layer = _Layer(block, attention)
    rn = lambda: torch.randn(2, 128, 256, device=DEV, dtype=BF)  # noqa: E731
    xs, ups = [rn().requires_grad_(True) for _ in range(4)], [rn() for _ in range(4)]
    exact = ["mlp.fc1.weight", "mlp.fc2.weight"]
    params = dict(block.named_parameters())
    leaves = [params[k] for k in exact]

    def step(f, x, up):
        y = f(x)
        wanted = leaves if attention else [x, *leaves]
        every = [*wanted, *([params["attn.c_attn.weight"], x] if attention else [])]
        grads = torch.autograd.grad(y, every, up)
        return [y.detach().clone(), *[g.clone() for g in grads[:len(wanted)]]]
    want = [step(layer, x, u) for x, u in zip(xs, ups)]
    # (the sample becomes the graphs' own input, which every call overwrites)
    graphed = torch.cuda.make_graphed_callables(layer, (rn().requires_grad_(True),), allow_unused_input=not attention)
    for turn in range(2):  # each graph replayed with eager work and the other inputs between
        for x, u, e in zip(xs, ups, want):
            got = step(graphed, x, u)
            torch.cuda.synchronize()
            same = [torch.equal(a, b) for a, b in zip(got, e)]
            assert all(same), (turn, same)
