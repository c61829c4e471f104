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


def test_no_full_projection_weights_are_held():
    m = model(d_model=96, bias=True)
    m8 = served(m)
    c = m.config
    full = {2 * c.d_inner * c.d_model, c.d_inner * c.d_model}
    for name, t in m8.state_dict().items():
        assert t.dtype == torch.int8 or t.numel() not in full, name
    assert not any(p.numel() in full for p in m8.parameters())
    # neither does a conversion of what is served reach the model, nor training it what is served
    x = torch.randn(2, 9, 96, device=DEV)
    y = m8(x)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(1)
    assert torch.equal(m8(x), y)
    m8.bfloat16()
    assert all(p.dtype == torch.float32 for p in m.parameters())


@pytest.mark.parametrize("d_model", [75, 96])
def test_copies_keep_the_rows_alignment(d_model, monkeypatch):
    """d_model 75: rows of 75 and 150 values.  No product copies its weight first, before
    or after the module has been copied, saved and loaded."""
    import copy

    from momentummamba_b200 import int8
    m = model(d_model=d_model, n_layers=1)
    x = torch.randn(2, 9, d_model, device=DEV)
    first = served(m)
    y = first(x)
    clone = copy.deepcopy(first).cpu().to(DEV)
    loaded = served(model(d_model=d_model, n_layers=1, seed=5))
    loaded.load_state_dict({k: v.clone() for k, v in first.state_dict().items()})
    taken = []
    rows = int8._tma_rows
    monkeypatch.setattr(int8, "_tma_rows", lambda t: taken.append((t, rows(t))) or taken[-1][1])
    for m8 in (first, clone, loaded):
        assert torch.equal(m8(x), y)
    assert len(taken) == 3 * 4 and all(out[2] is t for t, out in taken)
