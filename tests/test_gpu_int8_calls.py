"""How the 8-bit operators are called: types of weights, calls without a gradient."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_a_16_bit_norm_weight(dtype):
    """Converted to fp32 for the kernels: outputs and gradients are those of its fp32 values,
    the weight's own rounded once to its type."""
    from momentummamba_b200 import int8
    g = torch.Generator(device=DEV).manual_seed(1)
    x, dn = torch.randn(300, 264, generator=g, device=DEV), torch.randn(300, 264, generator=g, device=DEV)
    w16 = (1 + 0.2 * torch.randn(264, generator=g, device=DEV)).to(dtype).requires_grad_()
    w32 = w16.detach().float().requires_grad_()
    outs = []
    for w in (w16, w32):
        xi = x.clone().requires_grad_()
        n, _ = int8.rms_norm_ckpt(xi, w)
        outs.append((n, *torch.autograd.grad(n, [xi, w], dn)))
    (n16, dx16, dw16), (n32, dx32, dw32) = outs
    assert torch.equal(n16, n32) and torch.equal(dx16, dx32)
    assert dw16.dtype == dtype and torch.equal(dw16, dw32.to(dtype))
