"""weight_grad_ckpt against 64-bit products with what the checkpoint kept.

Tolerance, for S = sum of |terms| of a result: the tensor cores add 16 terms a
step into an fp32 accumulator, each step off by at most 2^-23 of a partial sum
that S bounds; slices of the tokens add one such step each (148 at most).
Products with 16-bit dy are exact, unless a row factor makes the kept value
round to dy's type (ULP of each term); fp32 dy carries 24 bits in three parts
(three steps for one) and one more rounding with a row factor.  The result's own
rounding comes last.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(M, N, K, dtype, seed=0, pad=0):
    g = torch.Generator(device=DEV).manual_seed(seed * 65537 + M * 131 + N * 17 + K)
    x = (torch.randn(M, K, generator=g, device=DEV) * torch.exp(torch.randn(K, generator=g, device=DEV))).to(dtype)
    dy = torch.randn(M, N + pad, generator=g, device=DEV).to(dtype)[:, :N]
    row = torch.rand(M, generator=g, device=DEV) + 0.5
    col = 1 + 0.2 * torch.randn(K, generator=g, device=DEV)
    return x, dy, row, col


def check(dw, dy, kept, row, col, dtype):
    M = dy.shape[0]
    kept, dy64 = kept.double(), dy.double()
    if row is not None:
        kept = kept * row.double()[:, None]
    want, size = dy64.t() @ kept, dy64.abs().t() @ kept.abs()
    if col is not None:
        want, size = want * col.double(), size * col.double().abs()
    parts = 3 if dy.dtype == torch.float32 else 1
    rel = (parts * -(-M // 16) + 150) * 2.0 ** -23
    rel += 4 * 2.0 ** -24 if parts == 3 else (1.01 * ULP[dy.dtype] if row is not None else 0)
    # fp16 kept values below 2^-14 are multiples of 2^-24
    floor = dy64.abs().sum(0)[:, None] * TINY[dy.dtype] * 2 if row is not None else 0
    err = (dw.double() - want).abs()
    assert dw.dtype == dtype
    assert torch.all(err <= rel * size + 1.01 * ULP[dtype] * want.abs() + TINY[dtype] + floor), \
        f"largest error {float(err.max()):.3e} of {float(want.abs().max()):.3e}"


SIZES = [(1, 1, 1), (2, 8, 16), (15, 33, 130), (64, 256, 128), (65, 257, 129), (333, 777, 333),
         (1000, 64, 75), (4099, 130, 1000), (20000, 512, 128), (3000, 2048, 1024), (70, 4000, 2000)]


@pytest.mark.parametrize("normed", [False, True], ids=["plain", "normed"])
@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,N,K", SIZES, ids=lambda v: str(v))
def test_weight_grad(M, N, K, dtype, normed):
    from momentummamba_b200 import int8
    x, dy, row, col = make(M, N, K, dtype)
    ck = int8.checkpoint_rows(x)
    row, col = (row, col) if normed else (None, None)
    dw = int8.weight_grad_ckpt(dy, ck, row_scale=row, col_scale=col)
    assert dw.shape == (N, K)
    check(dw, dy, ck.restore(), row, col, dtype)
    assert torch.equal(dw, int8.weight_grad_ckpt(dy, ck, row_scale=row, col_scale=col))


@pytest.mark.parametrize("dy_type,out", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16),
                                         (torch.float16, torch.float32)])
def test_output_types_and_a_checkpoint_of_another_type(dy_type, out):
    from momentummamba_b200 import int8
    x, _, row, col = make(500, 200, 300, torch.float32)
    _, dy, _, _ = make(500, 200, 300, dy_type)
    ck = int8.checkpoint_rows(x)
    check(int8.weight_grad_ckpt(dy, ck, row, col, out_dtype=out), dy, ck.restore(), row, col, out)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
def test_strides_alignment_and_leading_dims(dtype):
    from momentummamba_b200 import int8
    M, N, K = 120, 72, 96
    x, dy, _, _ = make(M, N, K, dtype)
    ck = int8.checkpoint_rows(x.unflatten(0, (5, 24)))
    assert ck.shape == (5, 24, K)
    want = int8.weight_grad_ckpt(dy, ck)
    wide = torch.empty(M, N + 24, dtype=dtype, device=DEV)[:, 8:8 + N]     # aligned, strided
    odd = torch.empty(M, N + 3, dtype=dtype, device=DEV)[:, 1:1 + N]       # not aligned
    trans = torch.empty(N, M, dtype=dtype, device=DEV).t()
    for t in (wide, odd, trans):
        t.copy_(dy)
        assert torch.equal(int8.weight_grad_ckpt(t, ck), want)
    assert torch.equal(int8.weight_grad_ckpt(dy.unflatten(0, (5, 24)), ck), want)
    off = int8.Ckpt8(torch.empty(M * 101 + 3, dtype=torch.int8, device=DEV)[3:].view(M, 101)[:, :K].copy_(ck.q),
                     ck.scale)
    assert torch.equal(int8.weight_grad_ckpt(dy, off), want)


def test_one_gradient_against_differences():
    """d/dW of sum(dy * (kept @ W^T)) is linear in W: differences are exact up to
    rounding, whatever the step."""
    from momentummamba_b200 import int8
    M, N, K = 90, 20, 40
    x, dy, _, _ = make(M, N, K, torch.float32)
    ck = int8.checkpoint_rows(x)
    dw = int8.weight_grad_ckpt(dy, ck).double()
    kept, W = ck.restore().double(), torch.randn(N, K, device=DEV, dtype=torch.float64)
    loss = lambda w: (dy.double() * (kept @ w.t())).sum()
    S = (dy.double().abs().t() @ kept.abs())
    for seed in range(4):
        d = torch.randn(N, K, device=DEV, dtype=torch.float64,
                        generator=torch.Generator(device=DEV).manual_seed(seed))
        diff = (loss(W + d) - loss(W - d)) / 2
        assert abs((dw * d).sum() - diff) <= 200 * 2.0 ** -23 * (S * d.abs()).sum()


def test_no_rows_nans_and_streams():
    from momentummamba_b200 import int8
    x, dy, _, _ = make(0, 30, 40, torch.float32)
    dw = int8.weight_grad_ckpt(dy, int8.checkpoint_rows(x))
    assert dw.shape == (30, 40) and torch.all(dw == 0)
    # a NaN group reaches its own 128 columns and no others
    x, dy, _, _ = make(300, 40, 300, torch.bfloat16)
    x[100, 130] = float("nan")
    dw = int8.weight_grad_ckpt(dy, int8.checkpoint_rows(x))
    assert torch.isnan(dw[:, 128:256]).all()
    assert torch.isfinite(dw[:, :128]).all() and torch.isfinite(dw[:, 256:]).all()
    x, dy, row, col = make(5000, 700, 260, torch.float32)
    want = int8.weight_grad_ckpt(dy, int8.checkpoint_rows(x), row, col)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = int8.weight_grad_ckpt(dy + 0, int8.checkpoint_rows(x + 0), row + 0, col + 0)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


def test_refusals():
    from momentummamba_b200 import _lib, int8
    x, dy, row, col = make(20, 16, 32, torch.float32)
    ck = int8.checkpoint_rows(x)
    with pytest.raises(ValueError, match="checkpoint's 20 rows"):
        int8.weight_grad_ckpt(dy[:10], ck)
    with pytest.raises(ValueError, match="row_scale must hold 20"):
        int8.weight_grad_ckpt(dy, ck, row_scale=row[:5])
    with pytest.raises(ValueError, match="col_scale must hold 32"):
        int8.weight_grad_ckpt(dy, ck, col_scale=row)
    with pytest.raises(ValueError, match="fp32, bf16 or fp16"):
        int8.weight_grad_ckpt(dy.double(), ck)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        int8.weight_grad_ckpt(dy.cpu(), ck)
    lib = _lib.load()
    dw = torch.empty(16, 32, device=DEV)
    args = lambda ldd: (20, 16, 32, 0, dy.data_ptr(), ldd, ck.q.data_ptr(), ck.q.stride(0),
                        ck.scale.data_ptr(), None, None, 0, dw.data_ptr(), 32, None, None)
    assert lib.mmb_wgrad_ck8(*args(12)) == 2    # shorter than a row
    assert lib.mmb_wgrad_ck8(*args(18)) == 3    # not a multiple of 16 bytes
    big = (40000, 128, 128, 0, dy.data_ptr(), 128, ck.q.data_ptr(), 128, ck.scale.data_ptr(), None,
           None, 0, dw.data_ptr(), 128, None, None)
    assert lib.mmb_wgrad_ck8_work_floats(40000, 128, 128, 0) > 0
    assert lib.mmb_wgrad_ck8(*big) == 5         # several slices and no workspace: refused before any launch


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_values_at_the_types_own_limit(dtype):
    """Rows at the lowest value beside ordinary ones: finite products stay finite and exact."""
    from momentummamba_b200 import int8
    M, N, K = 130, 24, 160
    x, dy, _, _ = make(M, N, K, dtype)
    x[17] = torch.finfo(dtype).min
    x[40, 130:] = 1e36
    dy[17] = 0
    dy[40] *= 1e-30
    ck = int8.checkpoint_rows(x)
    check(int8.weight_grad_ckpt(dy, ck), dy, ck.restore(), None, None, dtype)
