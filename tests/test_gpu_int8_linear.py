"""linear_q8 against 64-bit products of the same integers and scales.

Tolerance: the sums are exact; converting one to fp32, two products with scales
and the bias' addition round four times, each to 2^-24 of a value no larger than
|sum * xs * ws| + |bias|; the output's own rounding is ULP of the result (and
TINY below fp16's normal range).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def rows8(rows, cols, seed, low=-127, high=127, pitch=None):
    from momentummamba_b200 import int8
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + rows * 31 + cols)
    pitch = pitch or (cols + 15) // 16 * 16
    # what lies past the rows' ends is not zero: it must not be read as data
    q = torch.full((rows, pitch), 77, dtype=torch.int8, device=DEV)[:, :cols]
    q.copy_(torch.randint(low, high + 1, (rows, cols), generator=g, device=DEV))
    scale = torch.rand(rows, generator=g, device=DEV) * 0.02 / cols ** 0.5 + 1e-4
    return int8.Q8Rows(q, scale)


def check(x, w, bias, dtype):
    from momentummamba_b200 import int8
    y = int8.linear_q8(x, w, bias, out_dtype=dtype)
    K = w.shape[1]
    s = (x.q.reshape(-1, K).double() @ w.q.double().t()) * x.scale.reshape(-1, 1).double() \
        * w.scale.double()
    want = s if bias is None else s + bias.double()
    size = s.abs() + (0 if bias is None else bias.double().abs())
    assert y.dtype == dtype and y.shape == (*x.shape[:-1], w.shape[0])
    err = (y.reshape(want.shape).double() - want).abs()
    assert torch.all(err <= 4 * 2.0 ** -24 * size + 1.01 * ULP[dtype] * want.abs() + TINY[dtype]), \
        f"largest error {float(err.max()):.3e} of {float(want.abs().max()):.3e}"


# the split kernel's token tiles, K slices with and without work, partial tiles in each dimension
SMALL = [(1, 128, 128), (1, 4096, 1024), (3, 40, 16), (16, 129, 300), (17, 512, 1), (31, 96, 1152),
         (48, 2048, 4096), (64, 1000, 777), (65, 130, 1160), (128, 257, 2048), (200, 700, 333),
         (1, 1, 1), (2, 9500, 4224)]
# the tile kernel's 128- and 256-channel tiles, several tiles a CTA, groups of token tiles
LARGE = [(1300, 1024, 256), (4096, 300, 130), (2500, 2000, 640), (9000, 1030, 96), (76800, 64, 40),
         (5000, 3000, 1100)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16],
                         ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,N,K", SMALL + LARGE, ids=lambda v: str(v))
def test_linear_q8(M, N, K, dtype):
    bias = torch.randn(N, device=DEV) if (M + N + K) % 2 else None
    check(rows8(M, K, 1), rows8(N, K, 2), bias, dtype)


@pytest.mark.parametrize("M,N,K", [(5, 33, 131071), (300, 2600, 131071)])
def test_largest_sums_do_not_overflow(M, N, K):
    from momentummamba_b200 import int8
    x, w = rows8(M, K, 1, -128, -128), rows8(N, K, 2, -128, -128)
    y = int8.linear_q8(x, w)
    want = 16384.0 * K * x.scale.double()[:, None] * w.scale.double()
    assert torch.all((y.double() - want).abs() <= 4 * 2.0 ** -24 * want)


def test_leading_dims_strides_and_alignment():
    from momentummamba_b200 import int8
    x, w = rows8(24, 80, 1), rows8(50, 80, 2)
    x3 = int8.Q8Rows(x.q.unflatten(0, (2, 3, 4)), x.scale.view(2, 3, 4))
    check(x3, w, None, torch.float32)
    y = int8.linear_q8(x, w)
    # rows off their boundaries, a transposed tensor, a wider pitch, a strided scale
    off = torch.empty(24 * 83 + 1, dtype=torch.int8, device=DEV)[1:].view(24, 83)[:, :80]
    off.copy_(x.q)
    tr = x.q.t().contiguous().t()
    wide = rows8(24, 80, 1, pitch=112).q
    wide.copy_(x.q)
    ss = torch.stack([x.scale, x.scale + 1], 1)[:, 0]
    for q in (off, tr, wide, x.q.contiguous()):
        assert torch.equal(int8.linear_q8(int8.Q8Rows(q, ss), w), y)
    one = int8.Q8Rows(x.q[0], x.scale[0])
    assert torch.equal(int8.linear_q8(one, w), y[0])


def test_zero_tokens_and_a_nan_scale():
    from momentummamba_b200 import int8
    w = rows8(50, 80, 2)
    y = int8.linear_q8(rows8(0, 80, 1), w)
    assert y.shape == (0, 50)
    x = int8.quantize_rows(torch.randn(300, 80, device=DEV).index_fill_(
        0, torch.tensor([7], device=DEV), float("nan")))
    y = int8.linear_q8(x, w)
    assert torch.isnan(y[7]).all() and torch.isfinite(y[:7]).all() and torch.isfinite(y[8:]).all()


def test_results_do_not_depend_on_the_stream():
    from momentummamba_b200 import int8
    x, w = rows8(700, 300, 1), rows8(400, 300, 2)
    y = int8.linear_q8(x, w, out_dtype=torch.bfloat16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x2 = int8.Q8Rows((x.q + 0).contiguous(), x.scale + 0)   # rows copied inside, on this stream
        y2 = int8.linear_q8(x2, w, out_dtype=torch.bfloat16)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, y2)


def test_refusals():
    from momentummamba_b200 import _lib, int8
    x, w = rows8(4, 64, 1), rows8(8, 64, 2)
    with pytest.raises(ValueError, match="share K"):
        int8.linear_q8(x, rows8(8, 65, 2))
    with pytest.raises(ValueError, match="bias must be"):
        int8.linear_q8(x, w, torch.zeros(7, device=DEV))
    with pytest.raises(ValueError, match="output type"):
        int8.linear_q8(x, w, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="131071"):
        int8.linear_q8(rows8(1, 131072, 1), rows8(1, 131072, 2))
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        int8.linear_q8(int8.Q8Rows(x.q.cpu(), x.scale.cpu()), w)
    lib = _lib.load()
    p = lambda t: t.data_ptr()
    out = torch.empty(4, 8, device=DEV)
    args = lambda ldx: (4, 8, 64, p(x.q), ldx, p(x.scale), p(w.q), 64, p(w.scale), None, 0, p(out),
                        8, None)
    assert lib.mmb_gemm_q8(*args(60)) == 2     # shorter than a row
    assert lib.mmb_gemm_q8(*args(72)) == 3     # not a multiple of 16
