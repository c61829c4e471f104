"""The 8-bit products called from host threads that have made no CUDA call before: a
serving thread, or autograd's own thread where the weight gradient comes first."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def in_new_thread(f):
    """f() in a thread of its own, after a first call here whose memory it finds cached."""
    want = f().clone()
    torch.cuda.synchronize()
    out = []

    def body():
        try:
            out.append(f())
        except Exception as e:      # raised again below, in the test's own thread
            out.append(e)

    t = threading.Thread(target=body)
    t.start()
    t.join()
    if isinstance(out[0], Exception):
        raise out[0]
    torch.cuda.synchronize()
    assert torch.equal(out[0], want)


@pytest.mark.parametrize("rows", [3, 20000])
def test_linear_from_a_new_thread(rows):
    from momentummamba_b200 import int8
    x, w = int8.quantize_rows(torch.randn(rows, 256, device=DEV)), int8.quantize_rows(torch.randn(384, 256, device=DEV))
    in_new_thread(lambda: int8.linear_q8(x, w))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_weight_gradient_from_a_new_thread(dtype):
    from momentummamba_b200 import int8
    ck = int8.checkpoint_rows(torch.randn(300, 200, device=DEV))
    dy = torch.randn(300, 64, device=DEV).to(dtype)
    in_new_thread(lambda: int8.weight_grad_ckpt(dy, ck))


def test_weight_gradient_first_in_the_autograd_thread():
    """Only the weight wants a gradient, so its kernel is the thread's first CUDA work
    (whichever test comes first in the process; the results agree in any order)."""
    from momentummamba_b200 import int8
    x, w = torch.randn(300, 200, device=DEV), torch.randn(64, 200, device=DEV, requires_grad=True)
    dy = torch.randn(300, 64, device=DEV)
    (dw,) = torch.autograd.grad(int8.linear_ckpt(x, w), w, dy)
    assert torch.equal(dw, int8.weight_grad_ckpt(dy, int8.checkpoint_rows(x)))
