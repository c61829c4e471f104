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
