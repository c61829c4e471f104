"""MambaMomentum served in 8 bits: the two large projections of every block on
linear_q8, their weights quantised once per output channel, their inputs per token.

    model8 = Int8MambaMomentum(model)          # model: a trained MambaMomentum
    y = model8(x)                              # (batch, length, d_model)
    y, caches = model8.step(x, caches)         # one token, caches as MambaMomentum.step's

Between the blocks only the residual stream is stored in full: each block adds
its predecessor's output to it, norms the sum and emits 8-bit rows in one kernel
(rms_norm_q8).  The conv, the scan and the two small projections (x_proj,
dt_proj: the recurrence's step sizes and B, C, which 8 bits would disturb most)
run as in the model.  What is served is a copy of the model as it is now: the
two projections in 8 bits alone, a quarter of their fp32 size, the rest in full.
Later changes to the model do not reach it, nor does .to() on it reach the model.
Blocks, norms, mixers and projections that have been replaced or hooked are
refused: their weights alone do not say what they compute.

No reference counterpart (the reference serves in fp32).  Inference only: no
gradients.
"""
from __future__ import annotations

import copy

import torch
import torch.nn as nn

from .conv import conv1d_step
from .int8 import Q8Rows, linear_q8, quantize_rows, rms_norm_q8
from .mamba_momentum import MambaMomentum, MambaMomentumBlock, ResidualBlock, RMSNorm, runs_as


def _ordinary(module, cls, name):
    if not runs_as(module, cls):
        raise ValueError(f"Int8MambaMomentum: {name} must be an ordinary {cls.__name__} without hooks, "
                         f"got {type(module).__name__} (merge adapters and remove hooks first)")
    return module


class Int8Linear(nn.Module):
    """A linear's weight as 8-bit rows (one scale an output channel) and its bias.

    Scales and bias are fp32 whatever type the module is moved to: .to(torch.bfloat16)
    or .half() changes what the model computes around the products, not the weights."""

    def __init__(self, linear: nn.Linear):
        super().__init__()
        w = quantize_rows(linear.weight.detach())
        # contiguous rows of a multiple of 16 bytes: copies and moves keep the alignment that
        # the product's loads need
        self.in_features = w.q.shape[1]
        self.register_buffer("q", nn.functional.pad(w.q, (0, -self.in_features % 16)))
        self.register_buffer("scale", w.scale)
        self.register_buffer("bias", None if linear.bias is None
                             else linear.bias.detach().float().clone())

    def _apply(self, fn, recurse=True):
        held = {"scale": self.scale, "bias": self.bias}
        super()._apply(fn, recurse)
        for name, old in held.items():
            new = getattr(self, name)
            if new is not None and new.dtype != torch.float32:
                setattr(self, name, old.to(new.device))
        return self

    def forward(self, x: Q8Rows, out_dtype: torch.dtype) -> torch.Tensor:
        q = self.q if self.q.shape[1] == self.in_features else self.q[:, :self.in_features]
        return linear_q8(x, Q8Rows(q, self.scale), self.bias, out_dtype=out_dtype)


class Int8Block(nn.Module):
    """One residual block; mixer holds what stays in full: all but the two projections."""

    def __init__(self, block: ResidualBlock):
        super().__init__()
        _ordinary(block, ResidualBlock, "a block")
        norm = _ordinary(block.norm, RMSNorm, "norm")
        mixer = _ordinary(block.mixer, MambaMomentumBlock, "mixer")
        _ordinary(mixer.in_proj, nn.Linear, "in_proj")
        _ordinary(mixer.out_proj, nn.Linear, "out_proj")
        self.norm = copy.deepcopy(norm)
        self.mixer = copy.deepcopy(mixer, {id(mixer.in_proj): None, id(mixer.out_proj): None})
        self.in_proj, self.out_proj = Int8Linear(mixer.in_proj), Int8Linear(mixer.out_proj)

    def _in(self, x, residual):
        if residual is not None and residual.dtype not in (x.dtype, torch.float32):
            residual = residual.float()  # a 16-bit input to an fp32 model: the stream widens
        n, h = rms_norm_q8(x, None if self.norm.use_mup else self.norm.weight, residual=residual,
                           eps=self.norm.eps)
        return self.in_proj(n, self.mixer.x_proj.weight.dtype), h

    def _out(self, y):
        return self.out_proj(quantize_rows(y), self.mixer.x_proj.weight.dtype)

    def forward(self, x, residual):
        xz, h = self._in(x, residual)
        return self._out(self.mixer.mix(xz)), h

    def step(self, x, residual, cache):
        h_state, v_state, inputs = cache
        xz, h = self._in(x, residual)
        x, z = xz.chunk(2, dim=1)
        conv = self.mixer.conv1d
        x, inputs = conv1d_step(x, inputs, conv.weight, conv.bias)
        y, h_state, v_state = self.mixer._ssm_step(x, h_state, v_state, z)
        return self._out(y), h, (h_state, v_state, inputs)


class Int8MambaMomentum(nn.Module):
    def __init__(self, model: MambaMomentum):
        super().__init__()
        self.config = model.config
        self.layers = nn.ModuleList([Int8Block(b) for b in model.layers])

    @torch.no_grad()
    def forward(self, x):
        h = None
        for layer in self.layers:
            x, h = layer(x, h)
        return x if h is None else x + h

    @torch.no_grad()
    def step(self, x, caches):
        """One token x (batch, d_model) through every layer; caches is updated in place."""
        h = None
        for i, layer in enumerate(self.layers):
            x, h, caches[i] = layer.step(x, h, caches[i])
        return (x if h is None else x + h), caches
