"""8-bit rows, 8-bit checkpoints and the norm's backward from them, against plain
64-bit restatements, at sizes where vector and single loads, one and several
warps a row, and partial groups meet.

Tolerances, derived from the arithmetic:
  * a stored value is rounded once to its type: half a unit in the last place,
    ULP = 2^-24 (fp32), 2^-8 (bf16), 2^-11 (fp16), plus fp32 arithmetic before it;
    fp16 values below 2^-14 are multiples of 2^-24: TINY = 2^-25 beside it;
  * sums over a row run in 32-value chains and trees of at most 9 levels:
    50 * 2^-24 = 3e-6 relative, half of that in rstd: R = 4e-6 covers both;
  * q is the nearest integer of an fp32 product: half a step and 127 * 2^-22;
  * dweight adds at most ~600 fp32 terms in a row (rows of one block, then the
    blocks' lines): 600 * 2^-24 = 4e-5 of the sum of magnitudes at worst.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
R = 4e-6
EPS = 1e-5
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(rows, cols, dtype, seed=0, pad=0):
    """Normal rows; pad > 0: rows cut out of wider ones (a stride of cols + pad)."""
    g = torch.Generator(device=DEV).manual_seed(seed * 1000003 + rows * 131 + cols)
    t = torch.randn(rows, cols + pad, generator=g, device=DEV) * 3
    return t.to(dtype)[:, :cols]


def rows64(h64, w64, norm=True, eps=EPS):
    rstd = 1 / torch.sqrt((h64 ** 2).mean(1, keepdim=True) + eps) if norm else 1.0
    v = h64 * (1 if w64 is None else w64)
    return v * rstd, v.abs().amax(1) * (rstd[:, 0] if norm else 1.0) / 127


def kept64(v, v64=None):
    """(q * s, s per value) of an 8-bit checkpoint of v (rows, cols), in 64 bits."""
    v = v.double()
    out, step = torch.empty_like(v), torch.empty_like(v)
    for a in range(0, v.shape[1], 128):
        part = v[:, a:a + 128]
        top = part.abs().amax(1, keepdim=True)
        s = torch.full_like(top, 2.0 ** -100)
        for e in range(-100, 130):
            s = torch.where(top > 127 * s, torch.full_like(s, 2.0 ** (e + 1)), s)
        out[:, a:a + 128] = torch.round(part / s) * s
        step[:, a:a + 128] = s
    return out, step


SIZES = [(1, 1), (1, 8), (3, 75), (5, 128), (4, 129), (7, 256), (9, 264), (6, 511), (33, 1000),
         (130, 1024), (2, 1032), (17, 2048), (3, 4104), (2, 8191), (2, 16384)]


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_norm_q8(rows, cols, dtype):
    from momentummamba_b200 import int8
    x, r = make(rows, cols, dtype, 1), make(rows, cols, dtype, 2)
    w = 1 + 0.2 * make(1, cols, torch.float32, 3)[0]
    out, h = int8.rms_norm_q8(x, w, residual=r, eps=EPS)
    assert out.q.shape == (rows, cols) and out.scale.shape == (rows,) and h.dtype == dtype
    h64 = x.double() + r.double()
    assert torch.all((h.double() - h64).abs() <= (1.01 * ULP[dtype] + 2.0 ** -24) * h64.abs())
    n64, s64 = rows64(h64, w.double())
    assert torch.all((out.scale.double() - s64).abs() <= R * s64)
    step = s64[:, None]
    assert torch.all((out.q.double() * step - n64).abs() <= (0.5 + 127 * 2.0 ** -22) * step)
    back = out.dequantize(dtype).double()
    assert torch.all((back - out.q.double() * step).abs()
                     <= (1.01 * ULP[dtype] + R) * (out.q.double() * step).abs() + step * R
                     + TINY[dtype])


@pytest.mark.parametrize("xt,rt", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32)])
@pytest.mark.parametrize("cols", [96, 333, 1024])
def test_norm_q8_with_an_fp32_residual_stream(xt, rt, cols):
    from momentummamba_b200 import int8
    x, r = make(12, cols, xt, 1), make(12, cols, rt, 2)
    out, h = int8.rms_norm_q8(x, None, residual=r, eps=EPS)
    assert h.dtype == rt
    h64 = x.double() + r.double()
    assert torch.all((h.double() - h64).abs() <= 2.0 ** -23 * h64.abs())
    n64, s64 = rows64(h64, None)
    assert torch.all((out.q.double() * s64[:, None] - n64).abs() <= 0.5001 * s64[:, None])


@pytest.mark.parametrize("pad", [0, 3, 8])
@pytest.mark.parametrize("cols", [64, 77, 640])
@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
def test_quantize_rows_strides_and_leading_dims(dtype, cols, pad):
    from momentummamba_b200 import int8
    x = make(24, cols, dtype, 4, pad).unflatten(0, (2, 3, 4))
    out = int8.quantize_rows(x)
    assert out.q.shape == x.shape and out.scale.shape == (2, 3, 4)
    v64, s64 = rows64(x.reshape(24, cols).double(), None, norm=False)
    assert torch.all((out.scale.reshape(-1).double() - s64).abs() <= 2.0 ** -23 * s64)
    q = out.q.reshape(24, cols).double()
    assert torch.all((q * s64[:, None] - v64).abs() <= 0.5001 * s64[:, None])
    assert torch.equal(q.abs().amax(1), torch.full((24,), 127.0, device=DEV, dtype=torch.float64))
    # a transposed tensor (no unit stride) and an expanded one
    t = make(cols, 24, dtype, 5).t()
    assert torch.equal(int8.quantize_rows(t).q, int8.quantize_rows(t.contiguous()).q)
    e = make(1, cols, dtype, 6).expand(5, cols)
    assert torch.equal(int8.quantize_rows(e).q, int8.quantize_rows(e.contiguous()).q)


def test_rows_of_zeros_infinities_nans_and_extremes():
    from momentummamba_b200 import int8
    x = make(8, 300, torch.float32, 7)
    x[0] = 0
    x[1, 17] = float("inf")
    x[2, 299] = float("nan")
    x[3] = 1e-42                          # denormals: below 2^-100, count as zero
    x[4, 5] = -3e38                       # its square is an infinity: the norm is zero
    x[5] = torch.finfo(torch.float32).min
    out = int8.quantize_rows(x)
    v = out.dequantize()
    assert torch.all(v[0] == 0) and torch.all(out.q[3] == 0)
    assert torch.isnan(v[1]).all() and torch.isnan(v[2]).all()
    assert torch.isfinite(v[[0, 3, 4, 5, 6, 7]]).all()
    assert torch.all(out.q[5] == -127)
    n, _ = int8.rms_norm_q8(x, eps=EPS)
    v = n.dequantize()
    assert torch.all(v[0] == 0) and torch.isnan(v[1]).all() and torch.isnan(v[2]).all()
    assert torch.all(v[4] == 0) and torch.isfinite(v[[0, 3, 4, 5, 6, 7]]).all()
    ck = int8.checkpoint_rows(x)
    k = ck.restore()
    assert torch.all(k[0] == 0) and torch.isfinite(k[[0, 3, 4, 5, 6, 7]]).all()
    assert torch.isnan(k[1, :128]).all() and torch.isfinite(k[1, 128:]).all()
    assert torch.isnan(k[2, 256:]).all() and torch.isfinite(k[2, :256]).all()


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_checkpoint_is_exact_to_its_definition(rows, cols, dtype):
    from momentummamba_b200 import int8
    x = make(rows, cols, dtype, 8) * torch.logspace(-6, 3, cols, device=DEV).to(dtype)
    ck = int8.checkpoint_rows(x)
    want, step = kept64(x)
    assert torch.equal(ck.restore(torch.float32).double(), want)   # powers of two: no rounding
    assert torch.equal(ck.scale.double(), step[:, ::128])
    assert ck.restore(dtype).dtype == dtype and ck.restore(dtype).shape == x.shape


def test_checkpoint_scale_at_its_edges():
    from momentummamba_b200 import int8
    top = torch.tensor([127.0, 127.00001, 63.5, 64.0, 1.984375, 1.9843751, 2.0, 1.0],
                       device=DEV)
    x = torch.zeros(8, 128, device=DEV)
    x[:, 77] = -top
    want, step = kept64(x)
    ck = int8.checkpoint_rows(x)
    assert torch.equal(ck.scale[:, 0].double(), step[:, 0])
    assert torch.equal(ck.restore().double(), want)


def backward64(dn, dh, w, kept, h64):
    cols = kept.shape[1]
    rstd = 1 / torch.sqrt((h64 ** 2).mean(1, keepdim=True) + EPS)
    z = kept * rstd
    g = dn * (1 if w is None else w)
    mean = (g * z).sum(1, keepdim=True) / cols
    dx = rstd * (g - z * mean) + (0 if dh is None else dh)
    size = rstd * (g.abs() + z.abs() * (g * z).abs().mean(1, keepdim=True)) + dx.abs()
    return dx, size, (dn * z).sum(0), (dn * z).abs().sum(0)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", SIZES + [(2399, 77), (5000, 256)])
def test_norm_ckpt_forward_and_gradients(rows, cols, dtype):
    from momentummamba_b200 import int8
    x, r = make(rows, cols, dtype, 1).requires_grad_(), make(rows, cols, dtype, 2).requires_grad_()
    w = (1 + 0.2 * make(1, cols, torch.float32, 3)[0]).requires_grad_()
    dn, dh = make(rows, cols, dtype, 4), make(rows, cols, dtype, 5)
    n, h = int8.rms_norm_ckpt(x, w, residual=r, eps=EPS)
    dx, dr, dw = torch.autograd.grad([n, h], [x, r, w], [dn, dh])
    h64 = x.detach().double() + r.detach().double()
    n64, _ = rows64(h64, w.detach().double())
    u = 1.01 * ULP[dtype]
    assert torch.all((n.double() - n64).abs() <= (u + R) * n64.abs() + TINY[dtype])
    assert torch.all((h.double() - h64).abs() <= (u + 2.0 ** -24) * h64.abs())
    kept, _ = kept64(x.detach().float() + r.detach().float())
    want, size, dw64, dwsize = backward64(dn.double(), dh.double(), w.detach().double(), kept, h64)
    assert torch.all((dx.double() - want).abs() <= u * want.abs() + 2 * R * size + TINY[dtype])
    assert torch.equal(dx, dr)
    assert torch.all((dw.double() - dw64).abs() <= 4e-5 * dwsize)


@pytest.mark.parametrize("xt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("nt", TYPES, ids=["f32", "bf16", "f16"])
def test_norm_ckpt_types_of_stream_and_output(xt, nt):
    """An fp32 residual stream, activations of one type and a norm of another."""
    from momentummamba_b200 import int8
    rows, cols = 21, 200
    x, r = make(rows, cols, xt, 1).requires_grad_(), make(rows, cols, torch.float32, 2).requires_grad_()
    w = (1 + 0.2 * make(1, cols, torch.float32, 3)[0]).requires_grad_()
    dn, dh = make(rows, cols, nt, 4), make(rows, cols, torch.float32, 5)
    n, h = int8.rms_norm_ckpt(x, w, residual=r, eps=EPS, out_dtype=nt)
    assert n.dtype == nt and h.dtype == torch.float32
    dx, dr, dw = torch.autograd.grad([n, h], [x, r, w], [dn, dh])
    assert dx.dtype == xt and dr.dtype == torch.float32 and dw.dtype == torch.float32
    h64 = x.detach().double() + r.detach().double()
    kept, _ = kept64(x.detach().float() + r.detach())
    want, size, dw64, dwsize = backward64(dn.double(), dh.double(), w.detach().double(), kept, h64)
    assert torch.all((dr.double() - want).abs() <= 2 * R * size)
    assert torch.all((dx.double() - want).abs() <= 1.01 * ULP[xt] * want.abs() + 2 * R * size
                     + TINY[xt])
    assert torch.all((dw.double() - dw64).abs() <= 4e-5 * dwsize)


def test_norm_ckpt_without_residual_weight_or_a_gradient():
    from momentummamba_b200 import int8
    x = make(40, 96, torch.float32, 1).requires_grad_()
    n, h = int8.rms_norm_ckpt(x, eps=EPS)
    assert h is x
    dn = make(40, 96, torch.float32, 2)
    (dx,) = torch.autograd.grad(n, x, dn)
    kept, _ = kept64(x.detach())
    want, size, _, _ = backward64(dn.double(), None, None, kept, x.detach().double())
    assert torch.all((dx.double() - want).abs() <= 2 * R * size)
    # only the sum's gradient: the norm's part is absent
    r = make(40, 96, torch.float32, 3).requires_grad_()
    w = torch.ones(96, device=DEV, requires_grad=True)
    n, h = int8.rms_norm_ckpt(x, w, residual=r, eps=EPS)
    dh = make(40, 96, torch.float32, 4)
    dx, dr = torch.autograd.grad(h, [x, r], dh)
    assert torch.equal(dx, dh) and torch.equal(dr, dh)
    # no gradient wanted: nothing is kept
    with torch.no_grad():
        n2, _ = int8.rms_norm_ckpt(x, w, residual=r, eps=EPS)
    assert torch.equal(n2, n) and not n2.requires_grad


def test_norm_ckpt_gradient_against_differences():
    """Central differences of the 64-bit norm along random directions.  The kept
    values are off by at most half a step e, so dx is off by at most
    rstd * (e' |mean(g z)| + |z| mean(|g| e')), e' = e * rstd (and a second-order
    term e' mean(|g| e')); differences of step t add t^2."""
    from momentummamba_b200 import int8
    rows, cols = 6, 160
    x, r = make(rows, cols, torch.float32, 11).requires_grad_(), make(rows, cols, torch.float32, 12)
    w = 1 + 0.2 * make(1, cols, torch.float32, 13)[0]
    dn, dh = make(rows, cols, torch.float32, 14), make(rows, cols, torch.float32, 15)
    n, h = int8.rms_norm_ckpt(x, w, residual=r, eps=EPS)
    (dx,) = torch.autograd.grad([n, h], [x], [dn, dh])

    def loss(x64):
        hh = x64 + r.double()
        return (rows64(hh, w.double())[0] * dn.double()).sum() + (hh * dh.double()).sum()

    x64 = x.detach().double()
    h64 = x64 + r.double()
    rstd = 1 / torch.sqrt((h64 ** 2).mean(1, keepdim=True) + EPS)
    _, step = kept64(x.detach() + r)
    e, z, g = 0.5 * step * rstd, h64 * rstd, dn.double() * w.double()
    off = rstd * (e * (g * z).mean(1, keepdim=True).abs() + (z.abs() + e) * (g.abs() * e).mean(1, keepdim=True))
    for seed in range(5):
        d = make(rows, cols, torch.float32, 20 + seed).double() / 3
        t = 1e-4
        diff = (loss(x64 + t * d) - loss(x64 - t * d)) / (2 * t)
        got = (dx.double() * d).sum()
        assert abs(got - diff) <= (off * d.abs()).sum() + 1e-5 * (dx.double() * d).abs().sum()


def test_results_repeat_and_follow_the_stream():
    from momentummamba_b200 import int8
    x, r = make(3000, 520, torch.bfloat16, 1).requires_grad_(), make(3000, 520, torch.bfloat16, 2)
    w = (1 + 0.2 * make(1, 520, torch.float32, 3)[0]).requires_grad_()
    dn = make(3000, 520, torch.bfloat16, 4)

    def once():
        n, h = int8.rms_norm_ckpt(x, w, residual=r, eps=EPS)
        return (n, h, *torch.autograd.grad(n, [x, w], dn))

    first = once()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = torch.zeros_like(x) + x.detach()          # made on the side stream just before
        out, _ = int8.rms_norm_q8(y, w.detach(), residual=r, eps=EPS)
        again = once()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    ref, _ = int8.rms_norm_q8(x.detach(), w.detach(), residual=r, eps=EPS)
    assert torch.equal(out.q, ref.q) and torch.equal(out.scale, ref.scale)


def test_no_rows():
    from momentummamba_b200 import int8
    x = torch.empty(0, 64, device=DEV, requires_grad=True)
    r = torch.empty(0, 64, device=DEV)
    w = torch.ones(64, device=DEV, requires_grad=True)
    out, h = int8.rms_norm_q8(x, w.detach(), residual=r)
    assert out.q.shape == (0, 64) and out.dequantize().shape == (0, 64) and h.shape == (0, 64)
    n, h = int8.rms_norm_ckpt(x, w, residual=r)
    dx, dw = torch.autograd.grad(n, [x, w], torch.empty_like(n))
    assert dx.shape == (0, 64) and torch.all(dw == 0)
    assert int8.checkpoint_rows(torch.empty(0, 5, 64, device=DEV)).restore().shape == (0, 5, 64)


def test_refusals():
    from momentummamba_b200 import int8
    x = make(4, 64, torch.float32)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        int8.rms_norm_q8(x.cpu())
    with pytest.raises(ValueError, match="fp32, bf16 or fp16"):
        int8.quantize_rows(x.double())
    with pytest.raises(ValueError, match="share a shape"):
        int8.rms_norm_q8(x, residual=x[:2])
    with pytest.raises(ValueError, match="x's type or fp32"):
        int8.rms_norm_ckpt(x, residual=x.bfloat16())
    with pytest.raises(ValueError, match="weight must be"):
        int8.rms_norm_q8(x, torch.ones(63, device=DEV))
    with pytest.raises(ValueError, match="not supported"):
        int8.checkpoint_rows(torch.zeros(2, int8.MAX_COLS + 1, device=DEV))
    with pytest.raises(ValueError, match="output type"):
        int8.quantize_rows(x).dequantize(torch.float64)
    with pytest.raises(ValueError, match="one scale a row"):
        int8.Q8Rows(x.to(torch.int8), torch.ones(3, device=DEV))
    with pytest.raises(ValueError, match="ceil"):
        int8.Ckpt8(x.to(torch.int8), torch.ones(4, 2, device=DEV))
