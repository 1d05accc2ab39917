"""The decoder's fused sublayers beside changed submodules: whatever is not the plain linear layer and rotation that the
operators stand for (a replaced module, a hook, a bias, a forward of its own) is called as it is."""

import pytest
import torch
from torch import nn

import attnres_decoder as AD
from oracle import attnres_oracle as O


class _Counting:
    """The oracle in the operators' place, counting calls."""

    def __init__(self):
        self.calls = []

    def qkv_norm_rotary(self, *args, **kw):
        self.calls.append("rotary")
        return O.qkv_norm_rotary_ref(*args, **kw)

    def swiglu_projection(self, *args):
        self.calls.append("swiglu")
        return O.swiglu_projection_ref(*args)


def _pair(change):
    """Fused and eager decoder of the same weights, both changed by `change(block)`; (outputs, calls, gradients)"""
    cfg = dict(n_layer=2, n_head=2, n_embd=16, mlp_hidden_dim=24, vocab_size=32, block_size=16, use_attnres=False)
    ops = _Counting()
    torch.manual_seed(1)
    fused = AD.Decoder(AD.DecoderConfig(**cfg, fuse_qkv_rotary=True, fuse_swiglu=True), ops=ops)
    eager = AD.Decoder(AD.DecoderConfig(**cfg))
    eager.load_state_dict(fused.state_dict())
    idx = torch.randint(0, 32, (2, 9))
    out = []
    for model in (fused, eager):
        blocks = [m for m in model.modules() if isinstance(m, AD.Block)]
        assert len(blocks) == 2
        torch.manual_seed(2)
        undo = change(blocks[1])
        y = model(idx, return_hidden=True)
        y.square().sum().backward()
        if undo is not None:
            undo.remove()
        out.append((y.detach(), [p.grad for p in model.parameters()]))
    for a, b in zip(out[0][1], out[1][1]):
        assert (a is None) == (b is None) and (a is None or torch.equal(a, b))
    assert torch.equal(out[0][0], out[1][0])
    return ops.calls


def test_plain_modules_take_the_operators():
    assert _pair(lambda block: None) == ["rotary", "swiglu"] * 2


class _Adapter(nn.Module):
    """A low-rank addition to a linear layer, as adapters make it: it has a weight, and more."""

    def __init__(self, base):
        super().__init__()
        self.weight = base.weight
        self.a = nn.Parameter(torch.randn(4, base.in_features) * 0.3)
        self.b = nn.Parameter(torch.randn(base.out_features, 4) * 0.3)

    def forward(self, x):
        return x @ self.weight.t() + x @ self.a.t() @ self.b.t()


class _Scaled(nn.Linear):
    def forward(self, x):
        return 2.0 * super().forward(x)


def _replace(make):
    def change(block):
        block.mlp.fc1 = make(block.mlp.fc1)
    return change


def _scaled(old):
    new = _Scaled(old.in_features, old.out_features, bias=False)
    new.weight = old.weight
    return new


def _biased(old):
    new = nn.Linear(old.in_features, old.out_features)
    new.weight = old.weight
    return new


def _own_forward(old):
    old.forward = lambda x, call=old.forward: 3.0 * call(x)
    return old


def _parametrized(old):
    class Half(nn.Module):
        def forward(self, w):
            return w / 2
    torch.nn.utils.parametrize.register_parametrization(old, "weight", Half())
    return old


def _global_hook(block):
    return torch.nn.modules.module.register_module_forward_hook(
        lambda m, args, out: out * 2.0 if isinstance(m, nn.Linear) and m.out_features == 48 else None)


CHANGES = {
    "adapter": _replace(_Adapter),
    "subclass": _replace(_scaled),
    "bias": _replace(_biased),
    "own_forward": _replace(_own_forward),
    "parametrized": _replace(_parametrized),
    "forward_hook": lambda block: block.mlp.fc1.register_forward_hook(lambda m, args, out: out + 1.0),
    "forward_pre_hook": lambda block: block.mlp.fc1.register_forward_pre_hook(lambda m, args: (args[0] * 0.5,)),
    "backward_hook": lambda block: block.mlp.fc1.register_full_backward_hook(lambda m, gi, go: (gi[0] * 2.0,)),
    "backward_pre_hook": lambda block: block.mlp.fc1.register_full_backward_pre_hook(lambda m, go: (go[0] * 2.0,)),
}


@pytest.mark.parametrize("name", sorted(CHANGES))
def test_a_changed_projection_is_called_as_it_is(name):
    assert _pair(CHANGES[name]) == ["rotary", "swiglu", "rotary"]


def test_hooks_on_every_module():
    assert _pair(_global_hook) == ["rotary", "rotary"]


def test_a_changed_rotation_is_called_as_it_is():
    class Slower(AD.RotaryEmbedding):
        def rotate(self, x):
            return super().rotate(x) * 0.5

    def subclass(block):
        old = block.attn.rope
        new = Slower(AD.DecoderConfig(n_head=2, n_embd=16, block_size=16))
        new.load_state_dict(old.state_dict())
        block.attn.rope = new

    def own(block):
        rope = block.attn.rope
        rope.rotate = lambda x, call=rope.rotate: call(x) * 0.5
    for change in (subclass, own):
        assert _pair(change) == ["rotary", "swiglu", "swiglu"]


def test_fused_sublayers_trace_whole():
    """torch.compile sees through the check of the modules: one graph, the operators in it."""
    cfg = AD.DecoderConfig(n_layer=1, n_head=2, n_embd=16, mlp_hidden_dim=24, vocab_size=32, block_size=16,
                           use_attnres=False, fuse_qkv_rotary=True, fuse_swiglu=True)
    ops = _Counting()
    torch.manual_seed(1)
    block = AD.Block(cfg, ops)
    x = torch.randn(2, 9, 16)
    want = block.feed_forward(block.attention(x)[0])[0]
    assert ops.calls == ["rotary", "swiglu"]
    torch._dynamo.reset()
    f = torch.compile(lambda t: block.feed_forward(block.attention(t)[0])[0], backend="eager", fullgraph=True)
    assert torch.equal(f(x), want)
