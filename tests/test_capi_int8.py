"""The 8-bit entry points refuse bad arguments before touching the device (no GPU
needed): every pointer here is made up and never dereferenced."""

import pytest

from momentummamba_b200 import _lib

OK, NULL, SHAPE, ALIGN, UNSUPPORTED, WORKSPACE = 0, 1, 2, 3, 4, 5
F32, BF16, F16 = 0, 1, 2
P = 4096  # 16-byte aligned


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def norm_q8(lib, rows=4, cols=64, xt=F32, x=P, ldx=64, rt=F32, res=None, ldr=64, h=None, ldh=64, q=P,
            ldq=64, scale=P):
    return lib.mmb_norm_q8(rows, cols, xt, x, ldx, rt, res, ldr, None, 1e-5, 1, h, ldh, q, ldq, scale,
                           None)


def test_norm_q8(lib):
    assert norm_q8(lib, rows=0) == OK                     # no work, no launch
    assert norm_q8(lib, rows=-1) == SHAPE
    assert norm_q8(lib, cols=0) == SHAPE
    assert norm_q8(lib, rows=2 ** 31) == SHAPE
    assert norm_q8(lib, cols=16385, ldx=16385, ldq=16400) == UNSUPPORTED
    assert norm_q8(lib, xt=3) == UNSUPPORTED
    assert norm_q8(lib, xt=BF16, rt=F16) == UNSUPPORTED   # a residual of another 16-bit type
    assert norm_q8(lib, xt=F32, rt=BF16) == UNSUPPORTED
    assert norm_q8(lib, x=None) == NULL
    assert norm_q8(lib, q=None) == NULL
    assert norm_q8(lib, scale=None) == NULL
    assert norm_q8(lib, ldx=63) == SHAPE
    assert norm_q8(lib, res=P, ldr=63) == SHAPE
    assert norm_q8(lib, h=P, ldh=63) == SHAPE
    assert norm_q8(lib, ldq=63) == SHAPE


def test_norm_ck8(lib):
    def fwd(rows=4, cols=64, n=P, nt=F32, q=P, scale=P):
        return lib.mmb_norm_ck8_fwd(rows, cols, F32, P, 64, F32, None, 64, None, 1e-5, 1, None, 64, nt,
                                    n, 64, q, 64, scale, None, None)

    assert fwd(rows=0) == OK
    assert fwd(scale=None) == NULL
    assert fwd(n=None, q=None) == NULL                     # nothing asked for
    assert fwd(nt=7) == UNSUPPORTED

    def bwd(rows=4, cols=64, dt=F32, xt=F32, dn=P, q=P, dx=P, dw=None, work=None, ld=64):
        return lib.mmb_norm_ck8_bwd(rows, cols, dt, dn, ld, xt, None, 64, None, q, 64, P, P, dx, 64, dw,
                                    work, None)

    assert bwd(rows=0) == OK
    assert bwd(dn=None) == NULL and bwd(q=None) == NULL and bwd(dx=None) == NULL
    assert bwd(dw=P) == WORKSPACE
    assert bwd(ld=60) == SHAPE
    assert bwd(dt=BF16, xt=F16) == UNSUPPORTED and bwd(dt=F32, xt=BF16) == UNSUPPORTED
    assert lib.mmb_norm_ck8_bwd_work_floats(0, 64) == 0
    assert lib.mmb_norm_ck8_bwd_work_floats(1000, 64) >= 64
    assert lib.mmb_norm_ck8_bwd_work_floats(1000, 16385) == 0


def test_gemm_q8(lib):
    def call(M=4, N=8, K=64, x=P, ldx=64, w=P, ldw=64, ot=F32, out=P, ldo=8, xs=P, ws=P):
        return lib.mmb_gemm_q8(M, N, K, x, ldx, xs, w, ldw, ws, None, ot, out, ldo, None)

    assert call(M=0) == OK
    assert call(M=-1) == SHAPE and call(N=0) == SHAPE and call(K=0) == SHAPE
    assert call(K=131072, ldx=131072, ldw=131072) == SHAPE  # its largest sum is 2^31
    assert call(x=None) == NULL and call(w=None) == NULL and call(out=None) == NULL
    assert call(xs=None) == NULL and call(ws=None) == NULL
    assert call(ldx=48) == SHAPE and call(ldw=48) == SHAPE and call(ldo=7) == SHAPE
    assert call(ldx=72) == ALIGN and call(x=P + 8) == ALIGN and call(w=P + 1) == ALIGN
    assert call(ot=5) == UNSUPPORTED


def test_wgrad_ck8(lib):
    def call(M=4, N=16, K=64, dt=F32, dy=P, ldd=16, q=P, ldq=64, scale=P, ot=F32, dw=P, ldw=64, work=None):
        return lib.mmb_wgrad_ck8(M, N, K, dt, dy, ldd, q, ldq, scale, None, None, ot, dw, ldw, work, None)

    assert call(M=-1) == SHAPE and call(N=0) == SHAPE and call(K=0) == SHAPE
    assert call(dt=3) == UNSUPPORTED and call(ot=-1) == UNSUPPORTED
    assert call(dy=None) == NULL and call(q=None) == NULL and call(scale=None) == NULL
    assert call(dw=None) == NULL
    assert call(ldd=12) == SHAPE and call(ldq=60) == SHAPE and call(ldw=63) == SHAPE
    assert call(ldd=18) == ALIGN and call(dt=BF16, ldd=20) == ALIGN and call(dy=P + 4) == ALIGN
    assert call(ldq=72) == ALIGN and call(q=P + 8) == ALIGN and call(work=P + 4) == ALIGN
    floats = lib.mmb_wgrad_ck8_work_floats(40000, 128, 128, F32)
    assert floats > 0 and floats % (128 * 128) == 0         # whole slices of the result
    assert lib.mmb_wgrad_ck8_work_floats(0, 128, 128, F32) == 0
    assert lib.mmb_wgrad_ck8_work_floats(8, 4096, 4096, BF16) == 0   # one slice


def test_restore_q8(lib):
    def call(rows=4, cols=64, q=P, ldq=64, scale=P, ot=F32, out=P, ldo=64):
        return lib.mmb_restore_q8(rows, cols, q, ldq, scale, 0, ot, out, ldo, None)

    assert call(rows=0) == OK
    assert call(cols=0) == SHAPE and call(ldq=63) == SHAPE and call(ldo=63) == SHAPE
    assert call(q=None) == NULL and call(scale=None) == NULL and call(out=None) == NULL
    assert call(ot=9) == UNSUPPORTED


def test_python_layer_refuses_cpu_tensors():
    import torch

    from momentummamba_b200 import int8
    x = torch.randn(4, 64)
    for call in (lambda: int8.rms_norm_q8(x), lambda: int8.quantize_rows(x),
                 lambda: int8.rms_norm_ckpt(x), lambda: int8.checkpoint_rows(x),
                 lambda: int8.linear_ckpt(x, torch.randn(8, 64)),
                 lambda: int8.norm_linear_ckpt(x, None, torch.randn(8, 64))):
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            call()
