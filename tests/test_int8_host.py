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
