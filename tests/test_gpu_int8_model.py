"""The 8-bit operators together: MambaMomentum trained with 8-bit checkpoints and
served as Int8MambaMomentum.

Tolerances:
  * forward with checkpoints: the same products on the same values; only the norm
    is another kernel's: fp32 rounding through two layers, 1e-5 of the largest value;
  * gradients with checkpoints: kept values are off by at most half a step, 1/128 of
    their group's largest value (4 standard deviations of normal values), uniformly:
    1/128 / sqrt(3) * 4 = 1.8e-2 of their size.  Two projections a block and two
    blocks add to 5e-2 of a gradient's norm at worst, its direction stays within
    cos >= 0.998;
  * served in 8 bits: against the same quantisation restated on fp64 products.  Both
    round the same values; where the two sums differ by fp32 rounding, a value on
    the edge of a step falls to either side (a fraction of about 1e-4 of them, by
    1/127 of the row's largest): 1e-3 of the output's norm;
  * and against the fp32 model: two 8-bit operands of up to 1.5e-2 relative error a
    product (as above), four products in a row: 6e-2 of the output's norm.
"""
import copy

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def model(act_ckpt="none", d_model=96, n_layers=2, bias=False, mup=False, seed=0):
    from momentummamba_b200.mamba_momentum import MambaMomentum, MambaMomentumConfig
    torch.manual_seed(seed)
    return MambaMomentum(MambaMomentumConfig(d_model=d_model, n_layers=n_layers, bias=bias, mup=mup,
                                             act_ckpt=act_ckpt)).to(DEV)


def twin(m, act_ckpt):
    t = copy.deepcopy(m)
    t.config.act_ckpt = act_ckpt
    for layer in t.layers:
        layer.mixer.config.act_ckpt = act_ckpt
    return t


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("d_model,bias,mup,shape", [(96, False, False, (3, 65)), (128, True, False, (2, 200)),
                                                    (75, True, False, (2, 33)), (64, False, True, (4, 40))])
def test_training_with_8_bit_checkpoints(d_model, bias, mup, shape):
    m = model(d_model=d_model, bias=bias, mup=mup)
    m8 = twin(m, "int8")
    x = torch.randn(*shape, d_model, device=DEV)
    g = torch.randn(*shape, d_model, device=DEV)
    xa, xb = x.clone().requires_grad_(), x.clone().requires_grad_()
    ya, yb = m(xa), m8(xb)
    assert float((ya - yb).detach().abs().max()) <= 1e-5 * float(ya.detach().abs().max())
    ya.backward(g)
    yb.backward(g)
    assert rel(xb.grad, xa.grad) <= 5e-2
    for (name, pa), (_, pb) in zip(m.named_parameters(), m8.named_parameters()):
        assert pb.grad is not None and pb.grad.dtype == pa.grad.dtype, name
        assert rel(pb.grad, pa.grad) <= 5e-2, name
        assert float(F.cosine_similarity(pa.grad.flatten(), pb.grad.flatten(), 0)) >= 0.998, name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_training_under_autocast(dtype):
    """Both paths in mixed precision: their own 16-bit rounding comes on top (3e-2 and
    6e-2, as for the plain path against fp32)."""
    m = model()
    m8 = twin(m, "int8")
    x, g = torch.randn(2, 100, 96, device=DEV), torch.randn(2, 100, 96, device=DEV)
    for k in (m, m8):
        with torch.autocast("cuda", dtype=dtype):
            y = k(x)
        k.y = y.detach()
        (y.float() * g).sum().backward()
    assert m8.y.dtype == m.y.dtype and rel(m8.y, m.y) <= 2e-2
    for (name, pa), (_, pb) in zip(m.named_parameters(), m8.named_parameters()):
        assert pb.grad.dtype == torch.float32
        assert rel(pb.grad, pa.grad) <= 5e-2 + (6e-2 if dtype == torch.bfloat16 else 3e-2), name


def test_training_keeps_less_memory():
    """What one block keeps between the passes: the plain path holds h, the norm's output
    and out_proj's input in fp32; with checkpoints a byte a value of h and of that input."""
    B, L, d = 8, 512, 128
    m = model(d_model=d, n_layers=1)
    x = torch.randn(B, L, d, device=DEV, requires_grad=True)

    def kept(k):
        y = k(x)
        del y
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = k(x)
        return torch.cuda.memory_allocated() - before - y.numel() * 4

    saved = kept(m) - kept(twin(m, "int8"))
    rows = B * L
    # norm: at least two fp32 copies of (rows, d) against one byte; out_proj's input is also
    # the scan's output, kept by out_proj alone
    assert saved >= rows * d * (8 - 1.25) + rows * 2 * d * (4 - 1.25)


def fake_rows(v):
    top = v.abs().amax(-1, keepdim=True)
    return torch.round(v * (127 / top)) * (top / 127)


def restated(m, x):
    """Int8MambaMomentum on plain products: fp64 around the model's own conv and scan."""
    h, out = None, x
    for layer in m.layers:
        h = out if h is None else out + h
        h64 = h.double()
        v = h * layer.norm.weight
        top = v.abs().amax(-1, keepdim=True)
        rstd = 1 / torch.sqrt((h64 ** 2).mean(-1, keepdim=True) + layer.norm.eps)
        n = torch.round(v * (127 / top)).double() * top.double() / 127 * rstd
        lin = lambda a, w, b: (a @ fake_rows(w).double().t() + (0 if b is None else b.double())).float()
        y = layer.mixer.mix(lin(n, layer.mixer.in_proj.weight, layer.mixer.in_proj.bias))
        out = lin(fake_rows(y).double(), layer.mixer.out_proj.weight, layer.mixer.out_proj.bias)
    return out + h


@pytest.mark.parametrize("d_model,bias,shape", [(96, False, (3, 65)), (128, True, (2, 300)), (75, True, (2, 33))])
def test_serving_in_8_bits(d_model, bias, shape):
    from momentummamba_b200.mamba_momentum_int8 import Int8MambaMomentum
    m = model(d_model=d_model, bias=bias)
    m8 = Int8MambaMomentum(m)
    x = torch.randn(*shape, d_model, device=DEV)
    with torch.no_grad():
        y, y8, want = m(x), m8(x), restated(m, x)
    assert y8.shape == y.shape and y8.dtype == y.dtype and not y8.requires_grad
    assert rel(y8 - x, want - x) <= 1e-3
    assert rel(y8 - x, y - x) <= 6e-2


def test_decoding_steps_follow_the_sequence():
    """Token by token and all at once quantise the same rows: 1e-3 as above."""
    from momentummamba_b200.mamba_momentum_int8 import Int8MambaMomentum
    m = model()
    m8 = Int8MambaMomentum(m)
    B, L = 4, 12
    x = torch.randn(B, L, 96, device=DEV)
    y = m8(x)
    c = m.config
    caches = [(torch.zeros(B, c.d_inner, c.d_state, device=DEV), torch.zeros(B, c.d_inner, c.d_state, device=DEV),
               torch.zeros(B, c.d_inner, c.d_conv - 1, device=DEV)) for _ in range(c.n_layers)]
    steps = []
    for t in range(L):
        out, caches = m8.step(x[:, t], caches)
        steps.append(out)
    assert rel(torch.stack(steps, 1) - x, y - x) <= 1e-3


def test_serving_a_bf16_model():
    from momentummamba_b200.mamba_momentum_int8 import Int8MambaMomentum
    m = model(d_model=128)
    x = torch.randn(2, 64, 128, device=DEV)
    with torch.no_grad():
        y = m(x)
        y8 = Int8MambaMomentum(m.bfloat16())(x.bfloat16())
    assert y8.dtype == torch.bfloat16
    assert rel(y8.float() - x, y - x) <= 6e-2 + 3e-2     # bf16 activations on top


def test_refusals():
    from momentummamba_b200 import int8
    from momentummamba_b200.mamba_momentum import MambaMomentumConfig
    with pytest.raises(ValueError, match="act_ckpt must be"):
        MambaMomentumConfig(d_model=64, n_layers=1, act_ckpt="int4")
    x, w = torch.randn(4, 64, device=DEV), torch.randn(32, 64, device=DEV)
    with pytest.raises(ValueError, match="share K"):
        int8.norm_linear_ckpt(x, None, w[:, :60])
    with pytest.raises(ValueError, match="bias must be"):
        int8.linear_ckpt(x, w, torch.zeros(31, device=DEV))
    with pytest.raises(ValueError, match="fp32, bf16 or fp16"):
        int8.linear_ckpt(x, w.double())
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        int8.linear_ckpt(x.cpu(), w)
