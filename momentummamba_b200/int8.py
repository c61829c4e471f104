"""The 8-bit path of a block: serving with 8-bit rows and weights, training with
8-bit activation checkpoints, on the sm_100a kernels.

Serving.  ``rms_norm_q8`` adds the residual, norms and emits 8-bit rows in one
pass; ``quantize_rows`` emits them without the norm (weights: one scale per
output channel; any activation: one per token)::

    h = x + residual;  v = h * weight
    q = round(v * 127 / max|v|);   scale = max|v| / sqrt(mean(h^2) + eps) / 127

Training.  ``checkpoint_rows`` keeps a tensor in 8 bits: groups of 128 columns,
each with the smallest power of two s (at least 2^-100) with max|v| <= 127 s,
q = round(v / s), kept value q * s -- 1.03 bytes a value, the same on every run.
``rms_norm_ckpt`` is the norm with the residual's addition whose backward reads
such a checkpoint of the sum::

    n = h * rstd * weight                                   (forward, from h itself)
    z = kept * rstd;  g = dn * weight
    dx = dresidual = rstd * (g - z * mean(g * z)) + dh;   dweight = sum(dn * z)

The reference has no counterpart: it keeps and multiplies everything in fp32.
Sums, statistics and scales are fp32; results repeat bit for bit.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib

GROUP = 128        # columns of a checkpoint's group
MAX_COLS = 16384   # widest row of the row kernels

_TYPES = {torch.float32: _lib.MMB_F32, torch.bfloat16: _lib.MMB_BF16, torch.float16: _lib.MMB_F16}


def _type(t: torch.Tensor, what: str) -> int:
    code = _TYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{what} must be fp32, bf16 or fp16, got {t.dtype}")
    return code


def _out_type(dtype: torch.dtype) -> int:
    code = _TYPES.get(dtype)
    if code is None:
        raise ValueError(f"the output type must be fp32, bf16 or fp16, got {dtype}")
    return code


def _rows2(t: torch.Tensor) -> torch.Tensor:
    """(rows, cols) with unit-stride rows that do not overlap."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if (t.stride(1) != 1 and t.shape[1] != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _weight(weight: Optional[torch.Tensor], cols: int) -> Optional[torch.Tensor]:
    if weight is None:
        return None
    if weight.shape != (cols,):
        raise ValueError(f"weight must be ({cols},), got {tuple(weight.shape)}")
    weight = weight.detach()
    if weight.dtype != torch.float32 or not weight.is_contiguous():
        weight = weight.float().contiguous()
    return weight


def _call(name: str, on: torch.Tensor, *args) -> None:
    fn = getattr(_lib.load(), name)
    if on.device.index == torch.cuda.current_device():
        st = fn(*args, torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(on.device):
            st = fn(*args, torch.cuda.current_stream().cuda_stream)
    if st:
        _lib.check(st, name)


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _empty_q(rows: int, cols: int, device) -> torch.Tensor:
    """int8 rows that start on 16-byte boundaries."""
    pitch = (cols + 15) // 16 * 16
    q = torch.empty((rows, pitch), dtype=torch.int8, device=device)
    return q if pitch == cols else q[:, :cols]


def _check_rows(x: torch.Tensor, residual: Optional[torch.Tensor], what: str):
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what}: x must have a last dimension of one or more")
    if x.shape[-1] > MAX_COLS:
        raise ValueError(f"{what}: rows of more than {MAX_COLS} values are not supported, "
                         f"got {x.shape[-1]}")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"{what}: x and residual must share a shape, got {tuple(x.shape)} "
                             f"and {tuple(residual.shape)}")
        if residual.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{what}: the residual must be of x's type or fp32, got "
                             f"{residual.dtype} with x {x.dtype}")


class Q8Rows:
    """8-bit rows: q int8 (..., cols), scale fp32 (...); row r stands for q[r] * scale[r]."""

    __slots__ = ("q", "scale")

    def __init__(self, q: torch.Tensor, scale: torch.Tensor):
        if q.dtype != torch.int8 or scale.dtype != torch.float32:
            raise ValueError(f"Q8Rows: q must be int8 and scale fp32, got {q.dtype}, {scale.dtype}")
        if q.shape[:-1] != scale.shape:
            raise ValueError(f"Q8Rows: one scale a row is wanted, got q {tuple(q.shape)} and "
                             f"scale {tuple(scale.shape)}")
        self.q, self.scale = q, scale

    @property
    def shape(self):
        return self.q.shape

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values the rows stand for, contiguous, in dtype."""
        return _restore(self.q, self.scale, False, dtype)


class Ckpt8:
    """An 8-bit checkpoint: q int8 (rows, cols), scale fp32 (rows, ceil(cols / 128)) of
    powers of two, shape the kept tensor's shape."""

    __slots__ = ("q", "scale", "shape")

    def __init__(self, q: torch.Tensor, scale: torch.Tensor, shape=None):
        if q.dtype != torch.int8 or scale.dtype != torch.float32 or q.dim() != 2:
            raise ValueError("Ckpt8: q must be int8 (rows, cols) and scale fp32")
        if scale.shape != (q.shape[0], -(-q.shape[1] // GROUP)) or not scale.is_contiguous():
            raise ValueError(f"Ckpt8: scale must be a contiguous (rows, ceil(cols / {GROUP})) "
                             f"tensor, got {tuple(scale.shape)} for q {tuple(q.shape)}")
        self.q, self.scale = q, scale
        self.shape = q.shape if shape is None else shape

    def restore(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The kept values, contiguous, in dtype."""
        return _restore(self.q, self.scale, True, dtype).view(self.shape)


def _restore(q, scale, grouped, dtype):
    _lib.require_cuda(q, scale)
    code = _out_type(dtype)
    out = torch.empty(q.shape, dtype=dtype, device=q.device)
    q2 = _rows2(q)
    if out.numel():
        scale = scale.contiguous()
        cols = q2.shape[1]
        _call("mmb_restore_q8", q, q2.shape[0], cols, _p(q2), _ld(q2), _p(scale), int(grouped),
              code, _p(out), cols)
    return out


def _norm_q8(x, weight, residual, eps, norm, what):
    _lib.require_cuda(x, weight, residual)
    xt = _type(x, what + ": x")
    _check_rows(x, residual, what)
    cols = x.shape[-1]
    x2 = _rows2(x.detach())
    rows = x2.shape[0]
    w = _weight(weight, cols)
    h = r2 = None
    rt = xt
    if residual is not None:
        rt = _type(residual, what + ": residual")
        r2 = _rows2(residual.detach())
        h = torch.empty(x.shape, dtype=residual.dtype, device=x.device)
    q = _empty_q(rows, cols, x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    if rows:
        _call("mmb_norm_q8", x, rows, cols, xt, _p(x2), _ld(x2), rt, _p(r2),
              cols if r2 is None else _ld(r2), _p(w), eps, norm, _p(h), cols, _p(q), _ld(q),
              _p(scale))
    if x.dim() != 2:
        q = q.unflatten(0, x.shape[:-1]) if x.dim() > 2 else q[0]
    return Q8Rows(q, scale), h


def rms_norm_q8(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
                residual: Optional[torch.Tensor] = None, eps: float = 1e-5):
    """(8-bit rows of the root-mean-square norm of h = x + residual, h).

    x (..., cols) fp32, bf16 or fp16; residual of x's shape, in x's type or
    fp32, None for none; weight (cols,) or None.  h is a new tensor in the
    residual's type (x itself without a residual).  No gradient."""
    rows, h = _norm_q8(x, weight, residual, float(eps), 1, "rms_norm_q8")
    return rows, x if h is None else h


def quantize_rows(x: torch.Tensor) -> Q8Rows:
    """8-bit rows of x (..., cols): one scale a row.  No gradient."""
    return _norm_q8(x, None, None, 0.0, 0, "quantize_rows")[0]


def _tma_rows(t: torch.Tensor) -> torch.Tensor:
    """int8 (rows, cols) whose rows start on 16-byte boundaries: t itself where they do."""
    if (t.stride(1) == 1 or t.shape[1] == 1) and t.data_ptr() % 16 == 0 and (
            t.shape[0] == 1 or (t.stride(0) % 16 == 0 and t.stride(0) >= t.shape[1])):
        return t
    out = _empty_q(t.shape[0], t.shape[1], t.device)
    out.copy_(t)
    return out


def linear_q8(x: Q8Rows, w: Q8Rows, bias: Optional[torch.Tensor] = None,
              out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """x @ w^T (+ bias) of 8-bit rows: x (..., K), w (N, K) -> (..., N) in out_dtype.

    Sums are exact integers (K <= 131071), scaled in fp32 and rounded once.
    Rows that do not start on 16-byte boundaries (quantize_rows and rms_norm_q8
    make ones that do) are copied first.  No gradient."""
    xq, wq = x.q, w.q
    _lib.require_cuda(xq, x.scale, wq, w.scale, bias)
    code = _out_type(out_dtype)
    if wq.dim() != 2 or xq.dim() < 1 or xq.shape[-1] != wq.shape[1]:
        raise ValueError(f"linear_q8: x (..., K) and w (N, K) must share K, got {tuple(xq.shape)} "
                         f"and {tuple(wq.shape)}")
    N, K = wq.shape
    if not 1 <= K <= 131071 or N < 1:
        raise ValueError(f"linear_q8: K must be 1..131071 and N at least 1, got K {K}, N {N}")
    if bias is not None:
        if bias.shape != (N,):
            raise ValueError(f"linear_q8: bias must be ({N},), got {tuple(bias.shape)}")
        bias = bias.detach().float().contiguous()
    out = torch.empty((*xq.shape[:-1], N), dtype=out_dtype, device=xq.device)
    if xq.dim() != 2:
        xq = xq.reshape(-1, K)
    M = xq.shape[0]
    if M:
        xq, wq = _tma_rows(xq), _tma_rows(wq)
        xs, ws = x.scale.contiguous(), w.scale.contiguous()
        _call("mmb_gemm_q8", out, M, N, K, xq.data_ptr(), _ld16(xq), xs.data_ptr(), wq.data_ptr(),
              _ld16(wq), ws.data_ptr(), _p(bias), code, out.data_ptr(), N)
    return out


def _ld16(t: torch.Tensor) -> int:
    """Row stride for the tensor maps: one row has whichever multiple of 16 holds it."""
    return t.stride(0) if t.shape[0] > 1 else (t.shape[1] + 15) // 16 * 16


def _norm_ckpt(x, weight, residual, eps, norm, n_dtype, keep, what):
    """(n, h, q, scale, rstd) of one mmb_norm_ck8_fwd call; x and residual checked here."""
    _lib.require_cuda(x, weight, residual)
    xt = _type(x, what + ": x")
    _check_rows(x, residual, what)
    cols = x.shape[-1]
    x2 = _rows2(x)
    rows, dev = x2.shape[0], x.device
    w = _weight(weight, cols)
    h = r2 = n = q = scale = rstd = None
    rt = xt
    if residual is not None:
        rt = _type(residual, what + ": residual")
        r2 = _rows2(residual)
        h = torch.empty(x.shape, dtype=residual.dtype, device=dev)
    nt = 0
    if n_dtype is not None:
        nt = _out_type(n_dtype)
        n = torch.empty(x.shape, dtype=n_dtype, device=dev)
    if keep:
        q = _empty_q(rows, cols, dev)
        scale = torch.empty((rows, -(-cols // GROUP)), device=dev)
        if norm:
            rstd = torch.empty((rows,), device=dev)
    if rows:
        _call("mmb_norm_ck8_fwd", x, rows, cols, xt, _p(x2), _ld(x2), rt, _p(r2),
              cols if r2 is None else _ld(r2), _p(w), eps, norm, _p(h), cols, nt, _p(n), cols,
              _p(q), cols if q is None else _ld(q), _p(scale), _p(rstd))
    return n, h, q, scale, rstd


def checkpoint_rows(x: torch.Tensor) -> Ckpt8:
    """x (..., cols) kept in 8 bits (fp32, bf16 or fp16 in)."""
    _, _, q, scale, _ = _norm_ckpt(x.detach(), None, None, 0.0, 0, None, True, "checkpoint_rows")
    return Ckpt8(q, scale, x.shape)


def _norm_ckpt_bwd(dn, dh, weight, q, scale, rstd, shape, dx_dtype, want_dw):
    """(dx, dweight): dn (..., cols); dh in dx_dtype or None."""
    cols = shape[-1]
    dn2 = _rows2(dn)
    dh2 = None if dh is None else _rows2(dh)
    rows, dev = dn2.shape[0], dn.device
    w = _weight(weight, cols)
    dx = torch.empty(shape, dtype=dx_dtype, device=dev)
    dw = work = None
    if want_dw:
        dw = torch.empty((cols,), device=dev)
        work = torch.empty((_lib.load().mmb_norm_ck8_bwd_work_floats(rows, cols),), device=dev)
    _call("mmb_norm_ck8_bwd", dn, rows, cols, _TYPES[dn.dtype], _p(dn2), _ld(dn2),
          _TYPES[dx_dtype], _p(dh2), cols if dh2 is None else _ld(dh2), _p(w), _p(q), _ld(q),
          _p(scale), _p(rstd), _p(dx), cols, _p(dw), _p(work))
    return dx, dw


def _bwd_types(dn, dh, out_dtype):
    """The types the backward kernel takes: dx in dn's type or fp32."""
    dx_dtype = dn.dtype if out_dtype == dn.dtype else torch.float32
    if dh is not None and dh.dtype != dx_dtype:
        dh = dh.to(dx_dtype)
    return dh, dx_dtype


class RmsNormCkptFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, n_dtype):
        keep = any(ctx.needs_input_grad[:3])
        n, h, q, scale, rstd = _norm_ckpt(x, weight, residual, eps, 1, n_dtype, keep,
                                          "rms_norm_ckpt")
        ctx.save_for_backward(weight, q, scale, rstd)
        ctx.meta = (x.shape, x.dtype, None if residual is None else residual.dtype)
        ctx.set_materialize_grads(False)
        return (n, h) if h is not None else n

    @staticmethod
    def backward(ctx, dn, dh=None):
        weight, q, scale, rstd = ctx.saved_tensors
        shape, xdt, rdt = ctx.meta
        need_x, need_w, need_r = ctx.needs_input_grad[:3]
        dw = None
        if dn is None:
            dx = dh
        else:
            dh, dx_dtype = _bwd_types(dn, dh, rdt or xdt)
            dx, dw = _norm_ckpt_bwd(dn, dh, weight, q, scale, rstd, shape, dx_dtype,
                                    need_w and weight is not None)
        cast = lambda t, dt: None if t is None else t if t.dtype == dt else t.to(dt)
        return (cast(dx, xdt) if need_x else None,
                cast(dw, weight.dtype) if dw is not None else None,
                cast(dx, rdt) if need_r and rdt is not None else None, None, None)


def rms_norm_ckpt(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
                  residual: Optional[torch.Tensor] = None, eps: float = 1e-5,
                  out_dtype: Optional[torch.dtype] = None):
    """(n, h): the root-mean-square norm of h = x + residual, and h, with
    gradients for x, weight and residual.  Between the passes only an 8-bit
    checkpoint of h and one fp32 per row are kept.

    Arguments as in rms_norm_q8; n is in out_dtype (x's type by default), h in
    the residual's type (x itself without a residual)."""
    out = RmsNormCkptFn.apply(x, weight, residual, float(eps), out_dtype or x.dtype)
    return out if residual is not None else (out, x)


def _tma_grad(dy: torch.Tensor) -> torch.Tensor:
    """dy (rows, N) whose rows start on 16-byte boundaries: dy itself where they do."""
    dy = _rows2(dy)
    size = dy.element_size()
    if dy.data_ptr() % 16 == 0 and (dy.shape[0] == 1 or dy.stride(0) * size % 16 == 0):
        return dy
    unit = 16 // size
    out = torch.empty((dy.shape[0], (dy.shape[1] + unit - 1) // unit * unit), dtype=dy.dtype,
                      device=dy.device)[:, : dy.shape[1]]
    out.copy_(dy)
    return out


def _factor(t: Optional[torch.Tensor], n: int, what: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.numel() != n:
        raise ValueError(f"weight_grad_ckpt: {what} must hold {n} values, got {tuple(t.shape)}")
    return t.detach().reshape(-1).float().contiguous()


def weight_grad_ckpt(dy: torch.Tensor, kept: Ckpt8, row_scale: Optional[torch.Tensor] = None,
                     col_scale: Optional[torch.Tensor] = None,
                     out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The weight gradient (N, K) of a linear whose input was kept in 8 bits:

        dw[n, k] = col_scale[k] * sum_m dy[m, n] * row_scale[m] * kept[m, k]

    dy (..., N) fp32, bf16 or fp16 with kept's rows; row_scale (one a row) and
    col_scale (K,) are a norm's rstd and weight where the linear stands behind
    one.  In dy's type unless out_dtype says otherwise; sums are fp32."""
    _lib.require_cuda(dy, kept.q, kept.scale, row_scale, col_scale)
    code = _type(dy, "weight_grad_ckpt: dy")
    M, K = kept.q.shape
    if dy.dim() < 1 or dy.shape[-1] < 1 or dy.numel() != M * dy.shape[-1]:
        raise ValueError(f"weight_grad_ckpt: dy (..., N) must have the checkpoint's {M} rows, got "
                         f"{tuple(dy.shape)}")
    N = dy.shape[-1]
    row, col = _factor(row_scale, M, "row_scale"), _factor(col_scale, K, "col_scale")
    out_dtype = out_dtype or dy.dtype
    oc = _out_type(out_dtype)
    dw = torch.empty((N, K), dtype=out_dtype, device=dy.device)
    dy2, q = _tma_grad(dy.detach()), _tma_rows(kept.q)
    work = None
    floats = _lib.load().mmb_wgrad_ck8_work_floats(M, N, K, code)
    if floats:
        work = torch.empty((floats,), device=dy.device)
    unit = 16 // dy.element_size()
    _call("mmb_wgrad_ck8", dy, M, N, K, code, dy2.data_ptr(),
          dy2.stride(0) if M > 1 else -(-N // unit) * unit, q.data_ptr(), _ld16(q),
          kept.scale.data_ptr(), _p(row), _p(col), oc, dw.data_ptr(), K, _p(work))
    return dw
