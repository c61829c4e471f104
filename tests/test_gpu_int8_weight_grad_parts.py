"""weight_grad_ckpt where 16 bits do not hold an operand: behind a norm, dy times the
row's factor has more bits than its type, and fp16 does not hold what a checkpoint
may.  Both are multiplied in two bf16 parts.

Tolerance, for S = sum of |terms|: dy * row is rounded once in fp32 (2^-24); the high
part (8 bits) leaves less than 2^-8 of it, of which the low part leaves 2^-17; the tensor cores
add 16 terms a step, each step off by at most 2^-23 of a partial sum, two steps for 16
tokens, and slices of the tokens one step each (148 at most).  Rounded to 16 bits
between (up to 2^-8 or 2^-11 a term), a result of a few tokens is far outside.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def make(M, N, K, x_type, dy_type, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed * 65537 + M * 131 + N * 17 + K)
    x = (torch.randn(M, K, generator=g, device=DEV) * torch.exp(torch.randn(K, generator=g, device=DEV))).to(x_type)
    dy = torch.randn(M, N, generator=g, device=DEV).to(dy_type)
    row = torch.rand(M, generator=g, device=DEV) + 0.5
    col = 1 + 0.2 * torch.randn(K, generator=g, device=DEV)
    return x, dy, row, col


def products64(dy, kept, row, col):
    """(the gradient, the sum of its terms' sizes) in 64 bits."""
    a = dy.double() if row is None else dy.double() * row.double()[:, None]
    want, size = a.t() @ kept.double(), a.abs().t() @ kept.double().abs()
    return (want, size) if col is None else (want * col.double(), size * col.double().abs())


def two_parts(M):
    return (2 * -(-M // 16) + 150) * 2.0 ** -23 + 2.0 ** -17 + 2 * 2.0 ** -24


# one group and two groups a tile, one slice and several, whole and partial blocks
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (5, 24, 40), (33, 257, 129), (100, 700, 333), (64, 4096, 1024),
                                   (500, 200, 300), (700, 1032, 2000)], ids=lambda v: str(v))
def test_behind_a_norm_with_an_fp32_result(M, N, K, dtype):
    from momentummamba_b200 import int8
    x, dy, row, col = make(M, N, K, dtype, dtype)
    ck = int8.checkpoint_rows(x)
    dw = int8.weight_grad_ckpt(dy, ck, row, col, out_dtype=torch.float32)
    want, size = products64(dy, ck.restore(), row, col)
    assert torch.all((dw.double() - want).abs() <= two_parts(M) * size + 2.0 ** -23 * want.abs())
    assert torch.equal(dw, int8.weight_grad_ckpt(dy, ck, row, col, out_dtype=torch.float32))


def test_a_16_bit_result_is_rounded_once():
    """Over many tokens the result stands as near to 64 bits as rounding alone allows: a
    uniform error of half a unit in the last place, 2^-8 / (2 sqrt(3)) = 1.13e-3 of values
    at the low end of a binade and half of that at the high end, 0.82e-3..1.7e-3 over a
    normal distribution; an operand rounded to bf16 as well adds 1.6e-3 in square."""
    from momentummamba_b200 import int8
    x, dy, row, col = make(8192, 512, 256, torch.bfloat16, torch.bfloat16)
    ck = int8.checkpoint_rows(x)
    dw = int8.weight_grad_ckpt(dy, ck, row, col)
    want, _ = products64(dy, ck.restore(), row, col)
    ideal = float((want.bfloat16().double() - want).norm())
    assert dw.dtype == torch.bfloat16
    assert float((dw.double() - want).norm()) <= 1.01 * ideal


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_fp32_weights_under_autocast(dtype):
    """norm_linear_ckpt's own weight gradient: fp32 weights, a 16-bit product."""
    from momentummamba_b200 import int8
    M, N, K = 300, 64, 200
    x, dy, _, col = make(M, N, K, torch.float32, dtype)
    W = torch.randn(N, K, device=DEV, requires_grad=True)
    with torch.autocast("cuda", dtype=dtype):
        y, _ = int8.norm_linear_ckpt(x, col, W)
    assert y.dtype == dtype
    (dw,) = torch.autograd.grad(y, W, dy)
    rstd = 1 / torch.sqrt((x.double() ** 2).mean(1) + 1e-5)
    want, size = products64(dy, int8.checkpoint_rows(x).restore(), rstd, col)
    # the kernel's own rstd is off by 4e-6 at most
    assert dw.dtype == torch.float32
    assert torch.all((dw.double() - want).abs() <= (two_parts(M) + 4e-6) * size + 2.0 ** -23 * want.abs())


@pytest.mark.parametrize("normed", [False, True], ids=["plain", "normed"])
@pytest.mark.parametrize("scale", [1e-9, 1e-6, 1.0, 1e6], ids=str)
def test_fp16_gradients_with_a_checkpoint_beyond_fp16(scale, normed):
    """Kept fp32 values that fp16 does not hold (below 2^-25, beyond 65504): the products
    are what the formula says, in fp32 and, where the result fits, in fp16."""
    from momentummamba_b200 import int8
    M, N, K = 200, 40, 300
    x, dy, row, col = make(M, N, K, torch.float32, torch.float16)
    ck = int8.checkpoint_rows(x * scale)
    row, col = (row, col) if normed else (None, None)
    dw = int8.weight_grad_ckpt(dy, ck, row, col, out_dtype=torch.float32)
    want, size = products64(dy, ck.restore(), row, col)
    assert torch.all((dw.double() - want).abs() <= two_parts(M) * size + 2.0 ** -23 * want.abs())
    if scale == 1.0:
        half = int8.weight_grad_ckpt(dy, ck, row, col)
        assert torch.equal(half, dw.half())


def test_fp16_rows_at_the_types_own_limit():
    """A finite fp16 tensor beside masked rows of the lowest value: dy is 0 there, and the
    products stay finite."""
    from momentummamba_b200 import int8
    M, N, K = 130, 24, 160
    x, dy, _, _ = make(M, N, K, torch.float16, torch.float16)
    x[17] = torch.finfo(torch.float16).min
    x[40, 130:] = 65024.0
    dy[17] = 0
    dy[40] *= 1e-3
    ck = int8.checkpoint_rows(x)
    dw = int8.weight_grad_ckpt(dy, ck, out_dtype=torch.float32)
    want, size = products64(dy, ck.restore(), None, None)
    assert torch.isfinite(dw).all()
    assert torch.all((dw.double() - want).abs() <= two_parts(M) * size + 2.0 ** -23 * want.abs())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_an_fp32_result_over_many_tokens(dtype):
    """The sums leave the truncating accumulators every 4096 tokens.  Random terms: after i
    steps a partial sum has grown to sqrt(i / n) of its end; each step truncates up to 2^-23
    of it, 2^-24 on average, always towards zero.  n = 256 steps of one part add up to
    2 / 3 * 256 * 2^-24 = 1.0e-5 of a segment's sum, and independent segments' errors keep
    that ratio to their own sum; two parts take twice the steps."""
    from momentummamba_b200 import int8
    M, N, K = 65536, 4096, 1024
    g = torch.Generator(device=DEV).manual_seed(7)
    x = torch.randn(M, K, generator=g, device=DEV)
    dy = torch.randn(M, N, generator=g, device=DEV).to(dtype)
    ck = int8.checkpoint_rows(x)
    dw = int8.weight_grad_ckpt(dy, ck, out_dtype=torch.float32)
    kept = ck.restore().double()
    for cols in (slice(0, 64), slice(N - 64, N)):
        want = dy[:, cols].double().t() @ kept
        err = float((dw[cols].double() - want).norm() / want.norm())
        assert err <= (1.02e-5 if dtype == torch.bfloat16 else 2.04e-5)


@pytest.mark.parametrize("M,out,normed", [(9001, torch.float32, True), (9001, torch.float32, False),
                                          (40000, torch.bfloat16, True)], ids=str)
def test_sums_gathered_in_the_result_or_the_workspace(M, out, normed):
    """So many tiles that all tokens are one slice: an fp32 result gathers its segments in
    place, a 16-bit one in the workspace.  Without its last segment (809 or 7232 tokens) a
    result would be off by 20 and more, against a bound below 10."""
    from momentummamba_b200 import _lib, int8
    N, K = 8192, 8192
    assert (_lib.load().mmb_wgrad_ck8_work_floats(M, N, K, _lib.MMB_BF16) > 0) == (M > 32768)
    g = torch.Generator(device=DEV).manual_seed(M)
    x = torch.randn(M, K, generator=g, device=DEV).bfloat16()
    dy = torch.randn(M, N, generator=g, device=DEV).bfloat16()
    row = torch.rand(M, generator=g, device=DEV) + 0.5 if normed else None
    col = 1 + 0.2 * torch.randn(K, generator=g, device=DEV) if normed else None
    ck = int8.checkpoint_rows(x)
    del x
    dw = int8.weight_grad_ckpt(dy, ck, row, col, out_dtype=out)
    assert dw.dtype == out
    assert torch.equal(dw, int8.weight_grad_ckpt(dy, ck, row, col, out_dtype=out))
    kept = ck.restore(torch.bfloat16)
    for n, k in ((slice(0, 48), slice(0, 300)), (slice(N - 48, N), slice(K - 300, K)),
                 (slice(4000, 4048), slice(4000, 4300))):
        want, size = products64(dy[:, n], kept[:, k], row, None if col is None else col[k])
        bound = 2.0 ** -17 * size + 2.0 ** -8 * want.abs() * (out != torch.float32) + 2e-4 * M ** 0.5
        assert float(bound.max()) < 10
        assert torch.all((dw[n, k].double() - want).abs() <= bound)


def test_an_fp16_result_over_many_tokens_is_rounded_once():
    """So many tiles that all tokens are one slice: what the accumulators truncate before
    the sums leave them adds less than a hundredth to the result's own rounding."""
    from momentummamba_b200 import int8
    M, N, K = 65536, 8192, 8192
    g = torch.Generator(device=DEV).manual_seed(11)
    x = torch.randn(M, K, generator=g, device=DEV).half()
    dy = torch.randn(M, N, generator=g, device=DEV).half()
    ck = int8.checkpoint_rows(x)
    del x
    dw = int8.weight_grad_ckpt(dy, ck)
    want, _ = products64(dy[:, :64], ck.restore(torch.bfloat16)[:, :2048], None, None)
    ideal = float((want.half().double() - want).norm())
    assert float((dw[:64, :2048].double() - want).norm()) <= 1.01 * ideal
