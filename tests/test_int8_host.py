"""The host side of the 8-bit operators, without a GPU: what a call hands to the library.
The library's entry points are replaced by recorders; nothing is launched."""
import weakref

import pytest
import torch

from momentummamba_b200 import int8


@pytest.fixture
def calls(monkeypatch):
    """Names and arguments of the library calls made, on CPU tensors."""
    made = []
    monkeypatch.setattr(int8, "_index", lambda first, *others: 0)
    monkeypatch.setattr(int8, "_call", lambda name, idx, *args: made.append((name, args)))
    monkeypatch.setattr(int8, "_bwd_floats", lambda rows, cols: rows * cols)
    monkeypatch.setattr(int8._lib, "require_cuda", lambda *tensors: None)
    return made


def test_a_converted_norm_weight_lives_through_the_backward_call(calls, monkeypatch):
    """A norm weight that is not fp32 is converted; the copy must be held until the kernel
    that reads it is queued."""
    made, alive = [], []
    convert = int8._weight

    def tracked(weight, cols):
        w = convert(weight, cols)
        made.append(weakref.ref(w))
        return w

    monkeypatch.setattr(int8, "_weight", tracked)
    monkeypatch.setattr(int8, "_call", lambda name, idx, *args: alive.append(made[-1]() is not None))
    rows, cols = 4, 64
    q = int8._empty_q(rows, cols, "cpu")
    int8._norm_ckpt_bwd(torch.randn(rows, cols), None, torch.ones(cols, dtype=torch.bfloat16), q,
                        torch.zeros(rows * 2), torch.float32, True)
    assert alive == [True]


def kept(calls):
    """Whether each forward call was given a place for a checkpoint."""
    return [args[16] is not None for name, args in calls if name == "mmb_norm_ck8_fwd"]


@pytest.mark.parametrize("off", [torch.no_grad, torch.inference_mode], ids=["no_grad", "inference_mode"])
def test_no_checkpoint_where_no_gradient_is_wanted(calls, off):
    """Parameters that require a gradient, evaluated without one: the norm is called without
    a checkpoint, and the plain linear makes no library call at all."""
    x = torch.randn(4, 64)
    w, nw = torch.randn(8, 64, requires_grad=True), torch.ones(64, requires_grad=True)
    with off():
        n, _ = int8.rms_norm_ckpt(x, nw)
        y, _ = int8.norm_linear_ckpt(x, nw, w, residual=x)
        assert kept(calls) == [False, False]
        calls.clear()
        z = int8.linear_ckpt(x, w)
        assert calls == []
    assert not n.requires_grad and not y.requires_grad and not z.requires_grad


def test_checkpoints_where_a_gradient_is_wanted(calls):
    x = torch.randn(4, 64)
    w, nw = torch.randn(8, 64, requires_grad=True), torch.ones(64, requires_grad=True)
    b = torch.zeros(8, requires_grad=True)
    int8.rms_norm_ckpt(x, nw)
    int8.norm_linear_ckpt(x, nw, w)
    int8.linear_ckpt(x, w)
    assert kept(calls) == [True] * 3
    calls.clear()
    # frozen tensors, a frozen weight, only the bias trained: nothing reads a checkpoint
    int8.rms_norm_ckpt(x, nw.detach())
    int8.norm_linear_ckpt(x, nw.detach(), w.detach(), b)[0].sum().backward()
    int8.linear_ckpt(x.clone().requires_grad_(), w.detach())
    assert kept(calls) == [False] * 2 and torch.equal(b.grad, torch.full((8,), 4.0))


def test_a_block_takes_a_mixer_without_a_config():
    """A mixer replaced by any module: the block calls it, as it did before there were
    checkpoints."""
    from momentummamba_b200.mamba_momentum import MambaMomentumConfig, ResidualBlock
    block = ResidualBlock(MambaMomentumConfig(d_model=16, n_layers=1))
    block.mixer = torch.nn.Identity()
    x = torch.randn(2, 3, 16)
    assert torch.equal(block(x), block.norm(x) + x)


def test_the_model_imports_where_torch_has_no_cuda():
    """A torch built without CUDA lacks the stream and device entry points: models are
    still built, saved and loaded there."""
    import os
    import subprocess
    import sys
    code = ("import torch\n"
            "for name in [n for n in vars(torch._C) if n.startswith('_cuda_')]:\n"
            "    delattr(torch._C, name)\n"
            "from momentummamba_b200.mamba_momentum import MambaMomentum, MambaMomentumConfig\n"
            "import momentummamba_b200.mamba_momentum_int8, momentummamba_b200.LinOSS_pytorch\n"
            "MambaMomentum(MambaMomentumConfig(d_model=16, n_layers=1)).state_dict()\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True)
    assert run.returncode == 0, run.stderr[-2000:]
