"""Blocks whose modules have been replaced or hooked, trained with 8-bit checkpoints and
served in 8 bits: what a user put there runs, or is refused.

Tolerance of outputs: as in the model tests, 1e-5 of the largest value (the same
products; only the norm is another kernel's, in fp32); gradients 5e-2 of their norm
(kept values off by half a step)."""
import copy

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
PARTS = ["block", "norm", "mixer", "in_proj", "out_proj"]


def model(act_ckpt="none", seed=0):
    from momentummamba_b200.mamba_momentum import MambaMomentum, MambaMomentumConfig
    torch.manual_seed(seed)
    return MambaMomentum(MambaMomentumConfig(d_model=96, n_layers=3, act_ckpt=act_ckpt)).to(DEV)


def part(m, name, layer=1):
    block = m.layers[layer]
    return {"block": block, "norm": block.norm, "mixer": block.mixer, "in_proj": block.mixer.in_proj,
            "out_proj": block.mixer.out_proj}[name]


class Adapted(nn.Module):
    """A low-rank adapter around a linear that still shows its weight and bias."""

    def __init__(self, linear, rank=4):
        super().__init__()
        self.linear = linear
        self.a = nn.Parameter(0.3 * torch.randn(rank, linear.in_features, device=DEV))
        self.b = nn.Parameter(0.3 * torch.randn(linear.out_features, rank, device=DEV))

    weight = property(lambda self: self.linear.weight)
    bias = property(lambda self: self.linear.bias)

    def forward(self, x):
        return self.linear(x) + x @ self.a.t() @ self.b.t()


def compare(m, m8):
    x, g = torch.randn(2, 50, 96, device=DEV), torch.randn(2, 50, 96, device=DEV)
    y, y8 = m(x), m8(x)
    assert float((y8 - y).detach().abs().max()) <= 1e-5 * float(y.detach().abs().max())
    y.backward(g)
    y8.backward(g)
    for (name, a), (_, b) in zip(m.named_parameters(), m8.named_parameters()):
        assert float((b.grad - a.grad).norm()) <= 5e-2 * float(a.grad.norm()), name


@pytest.mark.parametrize("name", PARTS)
def test_hooks_run(name):
    m, m8 = model(), model("int8")
    seen = []
    part(m8, name).register_forward_hook(lambda mod, args, out: seen.append("forward"))
    part(m8, name).register_full_backward_hook(lambda mod, gin, gout: seen.append("backward"))
    compare(m, m8)
    assert seen == ["forward", "backward"]


@pytest.mark.parametrize("name", ["in_proj", "out_proj"])
def test_adapters_are_not_bypassed(name):
    m, m8 = model(), model("int8")
    torch.manual_seed(3)
    setattr(m.layers[1].mixer, name, Adapted(part(m, name)))
    setattr(m8.layers[1].mixer, name, copy.deepcopy(part(m, name)))
    compare(m, m8)


def test_a_replaced_norm_is_not_bypassed():
    m, m8 = model(), model("int8")
    for k in (m, m8):
        k.layers[1].norm = nn.LayerNorm(96).to(DEV)
    compare(m, m8)


def test_a_weight_computed_by_a_hook():
    """weight_norm sets the weight before each forward: a step on its parts changes it."""
    m, m8 = model(), model("int8")
    for k in (m, m8):
        nn.utils.weight_norm(k.layers[1].mixer.in_proj)
        with torch.no_grad():
            k.layers[1].mixer.in_proj.weight_g.mul_(1.5)
    compare(m, m8)


def test_a_parametrized_weight():
    class Twice(nn.Module):
        def forward(self, w):
            return 2 * w

    m, m8 = model(), model("int8")
    for k in (m, m8):
        nn.utils.parametrize.register_parametrization(k.layers[1].mixer.out_proj, "weight", Twice())
    compare(m, m8)


@pytest.mark.parametrize("name", PARTS)
def test_serving_refuses_what_its_weights_do_not_say(name):
    from momentummamba_b200.mamba_momentum_int8 import Int8MambaMomentum
    m = model()
    handle = part(m, name).register_forward_hook(lambda mod, args, out: None)
    with pytest.raises(ValueError, match="without hooks"):
        Int8MambaMomentum(m)
    handle.remove()
    Int8MambaMomentum(m)
    if name.endswith("proj"):
        setattr(m.layers[1].mixer, name, Adapted(part(m, name)))
        with pytest.raises(ValueError, match=f"{name} must be an ordinary Linear"):
            Int8MambaMomentum(m)
