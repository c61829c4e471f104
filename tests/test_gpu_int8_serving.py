"""Int8MambaMomentum: inputs, types and places that the model it serves takes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def model(d_model=96, n_layers=3, bias=False, seed=0):
    from momentummamba_b200.mamba_momentum import MambaMomentum, MambaMomentumConfig
    torch.manual_seed(seed)
    return MambaMomentum(MambaMomentumConfig(d_model=d_model, n_layers=n_layers, bias=bias)).to(DEV)


def served(m):
    from momentummamba_b200.mamba_momentum_int8 import Int8MambaMomentum
    return Int8MambaMomentum(m)


def caches(m, batch, dtype=torch.float32):
    c = m.config
    z = lambda n: torch.zeros(batch, c.d_inner, n, device=DEV, dtype=dtype)
    return [(z(c.d_state), z(c.d_state), z(c.d_conv - 1)) for _ in range(c.n_layers)]


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_16_bit_inputs_to_an_fp32_model(dtype):
    """The first block's input is 16 bits, the stream behind it fp32, as in the model: the
    same values given in fp32 take the same path (the norm widens what it reads)."""
    m = model()
    m8 = served(m)
    x = torch.randn(2, 40, 96, device=DEV).to(dtype)
    with torch.no_grad():
        want = m(x)
    y = m8(x)
    assert y.dtype == want.dtype == torch.float32
    assert torch.equal(y, m8(x.float()))
    ya, _ = m8.step(x[:, 0], caches(m, 2))
    yb, _ = m8.step(x[:, 0].float(), caches(m, 2))
    assert ya.dtype == torch.float32 and torch.equal(ya, yb)


def test_moving_to_another_type_leaves_the_8_bit_weights_alone():
    m = model(d_model=128, bias=True)
    x = torch.randn(2, 40, 128, device=DEV)
    with torch.no_grad():
        want = m(x)
    m8 = served(m)
    before = {k: v.clone() for k, v in m8.state_dict().items() if "proj" in k and "mixer" not in k}
    m8 = m8.to(torch.bfloat16)
    y = m8(x.bfloat16())
    assert y.dtype == torch.bfloat16
    assert rel(y.float() - x, want - x) <= 6e-2 + 3e-2    # 8 bits, and bf16 activations on top
    for back in (m8.half(), m8.float(), m8.cpu().to(DEV, torch.bfloat16)):
        after = back.state_dict()
        for k, v in before.items():
            assert after[k].dtype == v.dtype and torch.equal(after[k], v), k
