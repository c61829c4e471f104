"""The 8-bit operators at the limits of their types: what is finite stays finite."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("cols", [96, 128, 333, 520, 2048])
def test_fp16_checkpoints_restore_to_finite_fp16(cols):
    """A group of finite fp16 values is kept as finite fp16 values: the step is 1024 from
    65024 on, where 64 steps are 65536, so q stops at 63 there (off by one step at most)."""
    from momentummamba_b200 import int8
    x = torch.randn(6, cols, device=DEV).half()
    for i, top in enumerate((65504.0, -65504.0, 65472.0, 65024.0, 64992.0)):
        x[i, cols // 2] = top
    kept = int8.checkpoint_rows(x)
    half = kept.restore(torch.float16)
    assert torch.isfinite(half).all()
    assert torch.equal(half.float(), kept.restore(torch.float32))
    assert torch.all((half.double() - x.double()).abs() <= 1024)
    assert torch.all((half[4].double() - x[4].double()).abs() <= 256)     # step 512: ordinary rounding
    assert torch.all((half[5].double() - x[5].double()).abs() <= 2.0 ** -5)
    # the same through the norm, and with a residual in fp16; an fp32 sum may go beyond
    zero = torch.zeros_like(x)
    for res in (None, zero):
        q = int8._norm_ckpt(x, None, res, 1e-5, 1, torch.float16, True, "test")[2]
        assert torch.equal(q, kept.q)
    q = int8._norm_ckpt(x, None, zero.float(), 1e-5, 1, torch.float16, True, "test")[2]
    assert int(q[0, cols // 2]) == 64


TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("normed", [False, True], ids=["plain", "normed"])
@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
def test_weight_gradient_of_gradients_at_their_types_limit(dtype, normed):
    """dy of the type's lowest and largest value: against kept zeros it adds nothing, against
    small kept values what the formula says.

    Tolerance: at most 2 bf16 parts (2^-18 a term), steps of 2^-23 (3 parts, 16 tokens each,
    150 slices): (3 * 13 + 150) * 2^-23 + 2^-18 + 2^-24 = 2.7e-5 of the terms' sizes."""
    from momentummamba_b200 import int8
    M, N, K = 200, 24, 160
    g = torch.Generator(device=DEV).manual_seed(3)
    x, dy = torch.randn(M, K, generator=g, device=DEV), torch.randn(M, N, generator=g, device=DEV).to(dtype)
    x[17], dy[17] = 0, torch.finfo(dtype).min
    x[90], dy[90, :5] = x[90] * 1e-20, torch.finfo(dtype).max
    ck = int8.checkpoint_rows(x)
    row = torch.ones(M, device=DEV) if normed else None
    dw = int8.weight_grad_ckpt(dy, ck, row, out_dtype=torch.float32).double()
    kept = ck.restore().double()
    want, size = dy.double().t() @ kept, dy.double().abs().t() @ kept.abs()
    assert torch.isfinite(dw).all()
    assert torch.all((dw - want).abs() <= 2.7e-5 * size + 2.0 ** -23 * want.abs())


@pytest.mark.parametrize("normed", [False, True], ids=["plain", "normed"])
@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
def test_weight_gradient_of_infinite_gradients(dtype, normed):
    """An infinity in dy gives infinities of its sign (NaN against a kept zero) in its own
    row of the result and in no other."""
    from momentummamba_b200 import int8
    M, N, K = 200, 24, 160
    g = torch.Generator(device=DEV).manual_seed(4)
    x, dy = torch.randn(M, K, generator=g, device=DEV), torch.randn(M, N, generator=g, device=DEV).to(dtype)
    x[50, ::7] = 0
    dy[50, 3], dy[51, 9] = float("inf"), float("-inf")
    ck = int8.checkpoint_rows(x)
    row = torch.rand(M, generator=g, device=DEV) + 0.5 if normed else None
    dw = int8.weight_grad_ckpt(dy, ck, row, out_dtype=torch.float32).double()
    a = dy.double() if row is None else dy.double() * row.double()[:, None]
    want = (a[:, :, None] * ck.restore().double()[:, None, :]).sum(0)     # inf * 0 is NaN, term by term
    assert torch.equal(torch.isnan(dw), torch.isnan(want))
    assert torch.equal(dw[torch.isinf(want)], want[torch.isinf(want)])
    rest = [n for n in range(N) if n not in (3, 9)]
    assert torch.isfinite(dw[rest]).all()
