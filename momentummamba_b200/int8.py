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

``weight_grad_ckpt`` forms a linear's weight gradient from what its input's
checkpoint holds.  ``norm_linear_ckpt`` and ``linear_ckpt`` are the two layers
built of them: the norm's and the linear's backward share one checkpoint.

The reference has no counterpart: it keeps and multiplies everything in fp32.
Sums, statistics and scales are fp32; results repeat bit for bit.
"""
from __future__ import annotations

from functools import lru_cache
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib

GROUP = 128        # columns of a checkpoint's group
MAX_COLS = 16384   # widest row of the row kernels

_TYPES = {torch.float32: _lib.MMB_F32, torch.bfloat16: _lib.MMB_BF16, torch.float16: _lib.MMB_F16}

# A decoding step's kernels take a few microseconds, so its calls are held to a few
# too: the raw stream handle (torch.cuda.current_stream() builds an object, 3 us), one
# tensor for the small outputs of a call, sizes given one by one.
# A torch without CUDA has neither, and no call gets that far there.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_get_device = getattr(torch._C, "_cuda_getDevice", None)


def _type(t: torch.Tensor, what: str) -> int:
    code = _TYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{what}: tensors must be fp32, bf16 or fp16, got {t.dtype}")
    return code


def _out_type(dtype: torch.dtype) -> int:
    code = _TYPES.get(dtype)
    if code is None:
        raise ValueError(f"the output type must be fp32, bf16 or fp16, got {dtype}")
    return code


def _index(first: torch.Tensor, *others: Optional[torch.Tensor]) -> int:
    """The CUDA device that holds every given tensor; raises where there is none."""
    idx = first.get_device()
    for t in others:
        if t is not None and t.get_device() != idx:
            idx = -1
            break
    if idx < 0:
        _lib.require_cuda(first, *others)
    return idx


def _rows2(t: torch.Tensor) -> torch.Tensor:
    """(rows, cols) with unit-stride rows that do not overlap."""
    if t.dim() != 2:
        t = t.detach().reshape(-1, t.shape[-1])
    s0, s1 = t.stride()
    if (s1 != 1 or s0 < t.shape[1]) and ((s1 != 1 and t.shape[1] != 1)
                                         or (t.shape[0] > 1 and s0 < t.shape[1])):
        t = t.detach().contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _lines(t: torch.Tensor, cols: int):
    """(t as rows that the kernels take, their stride)."""
    if t.is_contiguous():
        return t, cols
    t = _rows2(t)
    return t, _ld(t)


def _like(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """A new contiguous tensor of t's shape."""
    if dtype == t.dtype and t.is_contiguous():
        return torch.empty_like(t, requires_grad=False)
    return torch.empty(t.shape, dtype=dtype, device=t.device)


def _weight(weight: Optional[torch.Tensor], cols: int) -> Optional[torch.Tensor]:
    if weight is None:
        return None
    if weight.dim() != 1 or weight.shape[0] != cols:
        raise ValueError(f"weight must be ({cols},), got {tuple(weight.shape)}")
    if weight.dtype != torch.float32 or weight.stride(0) != 1:
        weight = weight.detach().float().contiguous()
    return weight


_entry = {}


def _call(name: str, idx: int, *args) -> None:
    """One library call on the current stream of device idx."""
    fn = _entry.get(name)
    if fn is None:
        fn = _entry[name] = getattr(_lib.load(), name)
    if idx == _get_device():
        st = fn(*args, _raw_stream(idx))
    else:
        with torch.cuda.device(idx):
            st = fn(*args, _raw_stream(idx))
    if st:
        _lib.check(st, name)


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _empty_q(rows: int, cols: int, device) -> torch.Tensor:
    """int8 rows that start on 16-byte boundaries."""
    return torch.empty_strided((rows, cols), ((cols + 15) // 16 * 16, 1), dtype=torch.int8,
                               device=device)


def _check_rows(x: torch.Tensor, shape, residual: Optional[torch.Tensor], what: str) -> int:
    """The width of x's rows, checked with the residual's shape and type."""
    if not shape or shape[-1] < 1:
        raise ValueError(f"{what}: x must have a last dimension of one or more")
    cols = shape[-1]
    if cols > MAX_COLS:
        raise ValueError(f"{what}: rows of more than {MAX_COLS} values are not supported, "
                         f"got {cols}")
    if residual is not None:
        if residual.shape != shape:
            raise ValueError(f"{what}: x and residual must share a shape, got {tuple(shape)} "
                             f"and {tuple(residual.shape)}")
        rd = residual.dtype
        if rd is not torch.float32 and rd is not x.dtype:
            raise ValueError(f"{what}: the residual must be of x's type or fp32, got "
                             f"{rd} with x {x.dtype}")
    return cols


class Q8Rows:
    """8-bit rows: q int8 (..., cols), scale fp32 (...); row r stands for q[r] * scale[r]."""

    __slots__ = ("q", "scale")

    def __init__(self, q: torch.Tensor, scale: torch.Tensor):
        if q.dtype is not torch.int8 or scale.dtype is not torch.float32:
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


def _made(cls, q, scale):
    """Rows that a kernel has just made: nothing of them is left to check."""
    r = cls.__new__(cls)
    r.q, r.scale = q, scale
    return r


def _restore(q, scale, grouped, dtype):
    idx = _index(q, scale)
    code = _out_type(dtype)
    out = torch.empty(*q.shape, dtype=dtype, device=q.device)
    n = out.numel()
    if n:
        cols = q.shape[-1]
        q2, ldq = _lines(q, cols)
        scale = scale.contiguous()
        _call("mmb_restore_q8", idx, n // cols, cols, q2.data_ptr(), ldq, scale.data_ptr(), grouped,
              code, out.data_ptr(), cols)
    return out


def _norm_q8(x, weight, residual, eps, norm, what):
    idx = _index(x, weight, residual)
    xt = rt = _type(x, what)
    shape = x.shape
    cols = _check_rows(x, shape, residual, what)
    weight = _weight(weight, cols)
    x2, ldx = _lines(x, cols)
    rows, dev = x.numel() // cols, x.device
    h = rp = hp = None
    ldr = cols
    if residual is not None:
        rt = _TYPES[residual.dtype]
        r2, ldr = _lines(residual, cols)
        h = _like(residual, residual.dtype)
        rp, hp = r2.data_ptr(), h.data_ptr()
    q = _empty_q(rows, cols, dev)
    scale = torch.empty(rows, dtype=torch.float32, device=dev)
    if rows:
        _call("mmb_norm_q8", idx, rows, cols, xt, x2.data_ptr(), ldx, rt, rp, ldr, _p(weight),
              eps, norm, hp, cols, q.data_ptr(), q.stride(0), scale.data_ptr())
    if len(shape) != 2:
        q = q.unflatten(0, shape[:-1]) if len(shape) > 2 else q[0]
        scale = scale.view(shape[:-1])
    return _made(Q8Rows, q, scale), h


def rms_norm_q8(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
                residual: Optional[torch.Tensor] = None, eps: float = 1e-5):
    """(8-bit rows of the root-mean-square norm of h = x + residual, h).

    x (..., cols) fp32, bf16 or fp16; residual of x's shape, in x's type or
    fp32, None for none; weight (cols,) or None.  h is a new tensor in the
    residual's type (x itself without a residual).  No gradient."""
    rows, h = _norm_q8(x, weight, residual, eps, 1, "rms_norm_q8")
    return rows, x if h is None else h


def quantize_rows(x: torch.Tensor) -> Q8Rows:
    """8-bit rows of x (..., cols): one scale a row.  No gradient."""
    return _norm_q8(x, None, None, 0.0, 0, "quantize_rows")[0]


def _tma_rows(t: torch.Tensor):
    """(pointer, row stride, tensor) of int8 (rows, cols) whose rows start on 16-byte
    boundaries: t itself where they do, else a copy."""
    rows, cols = t.shape
    s0, s1 = t.stride()
    p = t.data_ptr()
    if (s1 == 1 or cols == 1) and not p & 15:
        if rows == 1:  # its stride says nothing: whichever multiple of 16 holds the row
            return p, (cols + 15) // 16 * 16, t
        if not s0 & 15 and s0 >= cols:
            return p, s0, t
    out = _empty_q(rows, cols, t.device)
    out.copy_(t)
    return out.data_ptr(), out.stride(0), out


def linear_q8(x: Q8Rows, w: Q8Rows, bias: Optional[torch.Tensor] = None,
              out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """x @ w^T (+ bias) of 8-bit rows: x (..., K), w (N, K) -> (..., N) in out_dtype.

    Sums are exact integers (K <= 131071), scaled in fp32 (by the token's scale, then
    the channel's) and rounded once.
    Rows that do not start on 16-byte boundaries (quantize_rows and rms_norm_q8
    make ones that do) are copied first.  No gradient."""
    xq, wq, xs, ws = x.q, w.q, x.scale, w.scale
    idx = _index(xq, xs, wq, ws, bias)
    code = _out_type(out_dtype)
    shape, wshape = xq.shape, wq.shape
    if len(wshape) != 2 or not shape or shape[-1] != wshape[1]:
        raise ValueError(f"linear_q8: x (..., K) and w (N, K) must share K, got {tuple(shape)} "
                         f"and {tuple(wshape)}")
    N, K = wshape
    if not 1 <= K <= 131071 or N < 1:
        raise ValueError(f"linear_q8: K must be 1..131071 and N at least 1, got K {K}, N {N}")
    bp = None
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != N:
            raise ValueError(f"linear_q8: bias must be ({N},), got {tuple(bias.shape)}")
        if bias.dtype != torch.float32 or bias.stride(0) != 1:
            bias = bias.detach().float().contiguous()
        bp = bias.data_ptr()
    if len(shape) == 2:
        M = shape[0]
        out = torch.empty(M, N, dtype=out_dtype, device=xq.device)
    else:
        out = torch.empty(*shape[:-1], N, dtype=out_dtype, device=xq.device)
        xq = xq.reshape(-1, K)
        M = xq.shape[0]
    if M:
        xp, ldx, xq = _tma_rows(xq)
        wp, ldw, wq = _tma_rows(wq)
        xs, ws = xs.contiguous(), ws.contiguous()
        _call("mmb_gemm_q8", idx, M, N, K, xp, ldx, xs.data_ptr(), wp, ldw, ws.data_ptr(), bp, code,
              out.data_ptr(), N)
    return out


def _norm_ckpt(x, weight, residual, eps, norm, n_dtype, keep, what):
    """(n, h, q, stats) of one mmb_norm_ck8_fwd call.  stats: the groups' scales and,
    with norm, one rstd a row behind them, in one fp32 tensor."""
    idx = _index(x, weight, residual)
    xt = rt = _type(x, what)
    cols = _check_rows(x, x.shape, residual, what)
    weight = _weight(weight, cols)
    x2, ldx = _lines(x, cols)
    rows, dev = x.numel() // cols, x.device
    h = n = q = stats = rp = hp = np_ = qp = sp = vp = None
    ldr = ldq = cols
    if residual is not None:
        rt = _TYPES[residual.dtype]
        r2, ldr = _lines(residual, cols)
        h = _like(residual, residual.dtype)
        rp, hp = r2.data_ptr(), h.data_ptr()
    nt = 0
    if n_dtype is not None:
        nt = _out_type(n_dtype)
        n = _like(x, n_dtype)
        np_ = n.data_ptr()
    if keep:
        groups = -(-cols // GROUP)
        q = _empty_q(rows, cols, dev)
        stats = torch.empty(rows * (groups + norm), dtype=torch.float32, device=dev)
        qp, ldq, sp = q.data_ptr(), q.stride(0), stats.data_ptr()
        vp = sp + 4 * rows * groups if norm else None
    if rows:
        _call("mmb_norm_ck8_fwd", idx, rows, cols, xt, x2.data_ptr(), ldx, rt, rp, ldr, _p(weight),
              eps, norm, hp, cols, nt, np_, cols, qp, ldq, sp, vp)
    return n, h, q, stats


def checkpoint_rows(x: torch.Tensor) -> Ckpt8:
    """x (..., cols) kept in 8 bits (fp32, bf16 or fp16 in)."""
    _, _, q, stats = _norm_ckpt(x, None, None, 0.0, 0, None, True, "checkpoint_rows")
    kept = _made(Ckpt8, q, stats.view(q.shape[0], -1) if q.shape[0] else
                 stats.view(0, -(-q.shape[1] // GROUP)))
    kept.shape = x.shape
    return kept


@lru_cache(maxsize=256)
def _bwd_floats(rows: int, cols: int) -> int:
    return _lib.load().mmb_norm_ck8_bwd_work_floats(rows, cols)


@lru_cache(maxsize=256)
def _wgrad_floats(M: int, N: int, K: int, code: int) -> int:
    return _lib.load().mmb_wgrad_ck8_work_floats(M, N, K, code)


def _norm_ckpt_bwd(dn, dh, weight, q, stats, out_dtype, want_dw):
    """(dx, dweight) from dn (..., cols): dx in out_dtype or, where the kernel has no
    such pair of types, fp32."""
    rows, cols = q.shape
    dev = dn.device
    idx = _index(dn, dh, weight, q)
    dx_dtype = dn.dtype if out_dtype == dn.dtype else torch.float32
    if dh is not None and dh.dtype != dx_dtype:
        dh = dh.to(dx_dtype)
    dn2, lddn = _lines(dn, cols)
    hp, lddh = None, cols
    if dh is not None:
        dh2, lddh = _lines(dh, cols)
        hp = dh2.data_ptr()
    dx = _like(dn, dx_dtype)
    dw = wp = kp = None
    if want_dw:
        dw = torch.empty(cols, dtype=torch.float32, device=dev)
        work = torch.empty(_bwd_floats(rows, cols), dtype=torch.float32, device=dev)
        wp, kp = dw.data_ptr(), work.data_ptr()
    weight = _weight(weight, cols)  # held until the call has been queued
    sp = stats.data_ptr()
    _call("mmb_norm_ck8_bwd", idx, rows, cols, _TYPES[dn.dtype], dn2.data_ptr(), lddn,
          _TYPES[dx_dtype], hp, lddh, _p(weight), q.data_ptr(), q.stride(0), sp,
          sp + 4 * rows * -(-cols // GROUP), dx.data_ptr(), cols, wp, kp)
    return dx, dw


def _grad_wanted(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether autograd records this call.  Read before a Function is applied: inside its
    forward grad mode is off, and needs_input_grad follows requires_grad alone."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _as(t: Optional[torch.Tensor], dtype) -> Optional[torch.Tensor]:
    return t if t is None or t.dtype == dtype else t.to(dtype)


def _backward_of(impl):
    """backward that impl computes once: a second derivative raises.  The wrapper that
    says so costs 6 us, and matters only where the backward itself is recorded."""
    guarded = once_differentiable(impl)

    def backward(ctx, *grads):
        return (guarded if torch.is_grad_enabled() else impl)(ctx, *grads)

    return staticmethod(backward)


def _rms_norm_ckpt_bwd(ctx, dn, dh=None):
    xdt, rdt = ctx.meta
    need_x, need_w, need_r = ctx.needs_input_grad[:3]
    weight, q, stats = ctx.saved_tensors
    dw = None
    if dn is None:
        dx = dh
    else:
        dx, dw = _norm_ckpt_bwd(dn, dh, weight, q, stats, rdt or xdt, need_w)
    return (_as(dx, xdt) if need_x else None, None if dw is None else _as(dw, weight.dtype),
            _as(dx, rdt) if need_r else None, None, None)


class RmsNormCkptFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, n_dtype):
        n, h, q, stats = _norm_ckpt(x, weight, residual, eps, 1, n_dtype,
                                    any(ctx.needs_input_grad[:3]), "rms_norm_ckpt")
        ctx.save_for_backward(weight, q, stats)
        ctx.meta = (x.dtype, None if residual is None else residual.dtype)
        ctx.set_materialize_grads(False)
        return (n, h) if h is not None else n

    backward = _backward_of(_rms_norm_ckpt_bwd)


def rms_norm_ckpt(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
                  residual: Optional[torch.Tensor] = None, eps: float = 1e-5,
                  out_dtype: Optional[torch.dtype] = None):
    """(n, h): the root-mean-square norm of h = x + residual, and h, with
    gradients for x, weight and residual.  Between the passes only an 8-bit
    checkpoint of h and one fp32 per row are kept.

    Arguments as in rms_norm_q8; n is in out_dtype (x's type by default), h in
    the residual's type (x itself without a residual)."""
    dt = out_dtype or x.dtype
    if not _grad_wanted(x, weight, residual):
        n, h, _, _ = _norm_ckpt(x, weight, residual, eps, 1, dt, False, "rms_norm_ckpt")
        return n, x if h is None else h
    out = RmsNormCkptFn.apply(x, weight, residual, eps, dt)
    return out if residual is not None else (out, x)


def _tma_grad(dy: torch.Tensor) -> torch.Tensor:
    """dy (rows, N) whose rows start on 16-byte boundaries: dy itself where they do."""
    dy = _rows2(dy)
    size = dy.element_size()
    if dy.data_ptr() % 16 == 0 and (dy.shape[0] == 1 or dy.stride(0) * size % 16 == 0):
        return dy
    unit = 16 // size
    out = torch.empty_strided(dy.shape, ((dy.shape[1] + unit - 1) // unit * unit, 1),
                              dtype=dy.dtype, device=dy.device)
    out.copy_(dy.detach())
    return out


def _factor(t: Optional[torch.Tensor], n: int, what: str) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.numel() != n:
        raise ValueError(f"weight_grad_ckpt: {what} must hold {n} values, got {tuple(t.shape)}")
    if t.dtype != torch.float32 or not t.is_contiguous():
        t = t.detach().float().contiguous()
    return t


def _weight_grad(idx, dy, code, q, scale_ptr, row_ptr, col_ptr, out_dtype, oc):
    M, K = q.shape
    N = dy.shape[-1]
    dw = torch.empty(N, K, dtype=out_dtype, device=dy.device)
    dy2 = _tma_grad(dy)
    qp, ldq, q = _tma_rows(q)
    floats = _wgrad_floats(M, N, K, code)
    work = torch.empty(floats, dtype=torch.float32, device=dy.device) if floats else None
    unit = 16 // dy.element_size()
    _call("mmb_wgrad_ck8", idx, M, N, K, code, dy2.data_ptr(),
          dy2.stride(0) if M > 1 else -(-N // unit) * unit, qp, ldq, scale_ptr, row_ptr, col_ptr, oc,
          dw.data_ptr(), K, _p(work))
    return dw


def weight_grad_ckpt(dy: torch.Tensor, kept: Ckpt8, row_scale: Optional[torch.Tensor] = None,
                     col_scale: Optional[torch.Tensor] = None,
                     out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The weight gradient (N, K) of a linear whose input was kept in 8 bits:

        dw[n, k] = col_scale[k] * sum_m dy[m, n] * row_scale[m] * kept[m, k]

    dy (..., N) fp32, bf16 or fp16 with kept's rows; row_scale (one a row) and
    col_scale (K,) are a norm's rstd and weight where the linear stands behind
    one.  In dy's type unless out_dtype says otherwise; sums are fp32."""
    q, scale = kept.q, kept.scale
    idx = _index(dy, q, scale, row_scale, col_scale)
    code = _type(dy, "weight_grad_ckpt")
    M, K = q.shape
    if dy.dim() < 1 or dy.shape[-1] < 1 or dy.numel() != M * dy.shape[-1]:
        raise ValueError(f"weight_grad_ckpt: dy (..., N) must have the checkpoint's {M} rows, got "
                         f"{tuple(dy.shape)}")
    row, col = _factor(row_scale, M, "row_scale"), _factor(col_scale, K, "col_scale")
    out_dtype = out_dtype or dy.dtype
    return _weight_grad(idx, dy, code, q, scale.data_ptr(), _p(row), _p(col), out_dtype,
                        _out_type(out_dtype))


def _linear_types(x_dtype: torch.dtype) -> torch.dtype:
    """The type a linear's product runs in: autocast's where it is on, else x's."""
    if torch.is_autocast_enabled("cuda"):
        return torch.get_autocast_dtype("cuda")
    return x_dtype


def _linear(n, weight, bias):
    dt = n.dtype
    with torch.autocast("cuda", enabled=False):
        return torch.nn.functional.linear(n, weight.to(dt), None if bias is None else bias.to(dt))


def _norm_linear_ckpt_bwd(ctx, dy, dh=None):
    xdt, rdt, bdt = ctx.meta
    need = ctx.needs_input_grad
    norm_weight, weight, q, stats = ctx.saved_tensors
    if dy is None:
        return _as(dh, xdt), None, _as(dh, rdt) if need[2] else None, None, None, None
    dx = dnw = dw = db = None
    if need[0] or need[1] or need[2]:
        with torch.autocast("cuda", enabled=False):
            dn = torch.matmul(dy, weight.to(dy.dtype))
        dx, dnw = _norm_ckpt_bwd(dn, dh, norm_weight, q, stats, rdt or xdt, need[1])
    if need[3]:
        rows, cols = q.shape
        sp, nw = stats.data_ptr(), _weight(norm_weight, cols)
        dw = _weight_grad(_index(dy, q, stats), dy, _TYPES[dy.dtype], q, sp,
                          sp + 4 * rows * -(-cols // GROUP), _p(nw), weight.dtype,
                          _out_type(weight.dtype))
    if need[4] and bdt is not None:
        db = dy.reshape(-1, dy.shape[-1]).sum(0, dtype=torch.float32).to(bdt)
    return (_as(dx, xdt) if need[0] else None,
            None if dnw is None else _as(dnw, norm_weight.dtype),
            _as(dx, rdt) if need[2] else None, dw, db, None)


class NormLinearCkptFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, norm_weight, residual, weight, bias, eps):
        dt = _linear_types(weight.dtype)
        n, h, q, stats = _norm_ckpt(x, norm_weight, residual, eps, 1, dt,
                                    any(ctx.needs_input_grad[:4]), "norm_linear_ckpt")
        y = _linear(n, weight, bias)
        ctx.save_for_backward(norm_weight, weight, q, stats)
        ctx.meta = (x.dtype, None if residual is None else residual.dtype,
                    None if bias is None else bias.dtype)
        ctx.set_materialize_grads(False)
        return (y, h) if h is not None else y

    backward = _backward_of(_norm_linear_ckpt_bwd)


def norm_linear_ckpt(x: torch.Tensor, norm_weight: Optional[torch.Tensor], weight: torch.Tensor,
                     bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                     eps: float = 1e-5):
    """(y, h): y = linear(rms_norm(h), weight, bias) of h = x + residual, and h.

    One 8-bit checkpoint of h serves both backward passes, the norm's and the
    weight's; neither h nor the norm is kept.  The product runs in the weight's
    type (autocast's where it is on); weight is (N, cols) fp32, bf16 or fp16."""
    _linear_check(x, weight, bias, "norm_linear_ckpt")
    if not _grad_wanted(x, norm_weight, residual, weight, bias):
        n, h, _, _ = _norm_ckpt(x, norm_weight, residual, eps, 1, _linear_types(weight.dtype), False,
                                "norm_linear_ckpt")
        return _linear(n, weight, bias), x if h is None else h
    out = NormLinearCkptFn.apply(x, norm_weight, residual, weight, bias, eps)
    return out if residual is not None else (out, x)


def _linear_ckpt_bwd(ctx, dy):
    xdt, bdt = ctx.meta
    need = ctx.needs_input_grad
    weight, q, stats = ctx.saved_tensors
    dx = dw = db = None
    if need[0]:
        with torch.autocast("cuda", enabled=False):
            dx = _as(torch.matmul(dy, weight.to(dy.dtype)), xdt)
    if need[1]:
        dw = _weight_grad(_index(dy, q, stats), dy, _TYPES[dy.dtype], q, stats.data_ptr(), None,
                          None, weight.dtype, _out_type(weight.dtype))
    if need[2] and bdt is not None:
        db = dy.reshape(-1, dy.shape[-1]).sum(0, dtype=torch.float32).to(bdt)
    return dx, dw, db


class LinearCkptFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        q = stats = None
        if ctx.needs_input_grad[1]:
            _, _, q, stats = _norm_ckpt(x, None, None, 0.0, 0, None, True, "linear_ckpt")
        ctx.save_for_backward(weight, q, stats)
        ctx.meta = (x.dtype, None if bias is None else bias.dtype)
        return _linear(x.to(_linear_types(weight.dtype)), weight, bias)

    backward = _backward_of(_linear_ckpt_bwd)


def linear_ckpt(x: torch.Tensor, weight: torch.Tensor,
                bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """linear(x, weight, bias) that keeps x in 8 bits for the weight's gradient."""
    _linear_check(x, weight, bias, "linear_ckpt")
    if not _grad_wanted(x, weight, bias):
        return _linear(x.to(_linear_types(weight.dtype)), weight, bias)
    return LinearCkptFn.apply(x, weight, bias)


def _linear_check(x, weight, bias, what):
    _lib.require_cuda(x, weight, bias)
    _type(weight, what)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what}: x (..., K) and weight (N, K) must share K, got {tuple(x.shape)} "
                         f"and {tuple(weight.shape)}")
    if bias is not None and (bias.dim() != 1 or bias.shape[0] != weight.shape[0]):
        raise ValueError(f"{what}: bias must be ({weight.shape[0]},), got {tuple(bias.shape)}")
