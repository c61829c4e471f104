"""The 8-bit operators on tensors of more than 2^31 values: rows at the far end equal
the same rows by themselves (the kernels treat rows alike wherever they lie), and the
weight gradient over all rows is the sum of its halves'.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
ROWS, COLS = 2 ** 21 + 4099, 1024          # 2^31 + 4.2e6 values


def test_rows_past_2_31_values():
    from momentummamba_b200 import int8
    x = torch.empty(ROWS, COLS, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    x[:4096] = torch.randn(4096, COLS, generator=g, device=DEV).bfloat16()
    for i in range(4096, ROWS, 4096):       # the same block again and again, scaled
        n = min(4096, ROWS - i)
        x[i:i + n] = x[:n] * (1 + (i // 4096) % 7)
    w = 1 + 0.1 * torch.randn(COLS, generator=g, device=DEV)
    tail = x[-300:].clone()
    out, _ = int8.rms_norm_q8(x, w)
    ref, _ = int8.rms_norm_q8(tail, w)
    assert torch.equal(out.q[-300:], ref.q) and torch.equal(out.scale[-300:], ref.scale)
    wq = int8.quantize_rows(torch.randn(1024, COLS, generator=g, device=DEV))
    y = int8.linear_q8(out, wq, out_dtype=torch.bfloat16)      # 2^31 results
    assert torch.equal(y[-300:], int8.linear_q8(ref, wq, out_dtype=torch.bfloat16))
    del y
    back = out.dequantize(torch.bfloat16)
    assert torch.equal(back[-300:], ref.dequantize(torch.bfloat16))
    del back, out
    n, h, q, stats = int8._norm_ckpt(x, w, None, 1e-5, 1, torch.bfloat16, True, "test")
    n1, _, q1, stats1 = int8._norm_ckpt(tail, w, None, 1e-5, 1, torch.bfloat16, True, "test")
    assert torch.equal(n[-300:], n1) and torch.equal(q[-300:], q1)
    dx, _ = int8._norm_ckpt_bwd(n, None, w, q, stats, torch.bfloat16, True)
    dx1, _ = int8._norm_ckpt_bwd(n1, None, w, q1, stats1, torch.bfloat16, True)
    assert torch.equal(dx[-300:], dx1)


def test_weight_gradient_past_2_31_values():
    """Halves added: each result's terms are the same, their order is not.  S = sum of
    |terms| <= sqrt(M) * norm of them; 2^21 / 16 steps of 2^-23 in at most 148 slices
    bound the difference by (2^21 / 16 / 2 + 300) * 2^-23 * S at the very worst; random
    rounding stays below its square root, 1e-4 of the largest result."""
    from momentummamba_b200 import int8
    g = torch.Generator(device=DEV).manual_seed(2)
    dy = torch.empty(ROWS, 1024, dtype=torch.bfloat16, device=DEV)
    x = torch.empty(ROWS, 128, dtype=torch.bfloat16, device=DEV)
    for i in range(0, ROWS, 2 ** 18):
        n = min(2 ** 18, ROWS - i)
        dy[i:i + n] = torch.randn(n, 1024, generator=g, device=DEV).bfloat16()
        x[i:i + n] = torch.randn(n, 128, generator=g, device=DEV).bfloat16()
    half = 2 ** 20
    dw = int8.weight_grad_ckpt(dy, int8.checkpoint_rows(x), out_dtype=torch.float32)
    parts = sum(int8.weight_grad_ckpt(dy[a:b], int8.checkpoint_rows(x[a:b]), out_dtype=torch.float32).double()
                for a, b in ((0, half), (half, ROWS)))
    assert float((dw.double() - parts).abs().max()) <= 1e-4 * float(parts.abs().max())
    # the far end counts: without its last rows the result is another
    tail = int8.weight_grad_ckpt(dy[-4099:], int8.checkpoint_rows(x[-4099:]), out_dtype=torch.float32)
    less = int8.weight_grad_ckpt(dy[:-4099], int8.checkpoint_rows(x[:-4099]), out_dtype=torch.float32)
    assert float((dw.double() - less.double() - tail.double()).abs().max()) <= 1e-4 * float(parts.abs().max())
