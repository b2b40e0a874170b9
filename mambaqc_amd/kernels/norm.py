"""Layer norm over the last axis, the norm before the head of the reference's LM (nn.LayerNorm,
models/quaternion_mamba2.py:79-81), with its gradients.

    h = (x - mean x) / sqrt(mean (x - mean x)^2 + eps),  y = h weight + bias
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .. import _native as nat

MAX_WIDTH = 8192  # elements of a row: sixteen in the registers of each of a workgroup's 512 lanes


def _check(x, weight, bias):
    if x.dim() < 1:
        raise ValueError("layer_norm: x has no axis to normalise")
    d = x.shape[-1]
    for name, w in (("weight", weight), ("bias", bias)):
        if w is not None and tuple(w.shape) != (d,):
            raise ValueError(f"layer_norm: {name} must be [{d}], got {tuple(w.shape)}")


def _operands(x, weight, bias):
    """The operands as the kernels read them, weights in fp32."""
    _check(x, weight, bias)
    return nat.host().LayerNorm(x, weight, bias, nat.param_f32)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm of x [..., d] over its last axis, times weight and plus bias ([d], either may be None), in
    x's dtype. Rows that are evenly spaced are read in place; means and sums are fp32. d is at most 8192.
    Differentiable in every tensor argument when autograd is recording (in reverse; forward mode is
    refused)."""
    if nat.compiling():
        _check(x, weight, bias)
        return torch.ops.mambaqc.layer_norm(x, weight, bias, eps)[0]
    y = nat.host().layer_norm(x, weight, bias, eps, nat.param_f32)
    if y is None:  # say what is wrong
        _check(x, weight, bias)
    return y


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm over the last axis, of at most 8192 elements, on the kernel (same parameters and state
    dict). The output is in the input's dtype, under autocast too."""

    def __init__(self, normalized_shape, eps: float = 1e-5, elementwise_affine: bool = True,
                 bias: bool = True, device=None, dtype=None):
        super().__init__(normalized_shape, eps, elementwise_affine, bias, device, dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError(f"LayerNorm: normalises over the last axis, got {self.normalized_shape}")
        if self.normalized_shape[0] > MAX_WIDTH:
            raise ValueError(f"LayerNorm: rows have at most {MAX_WIDTH} elements, got {self.normalized_shape[0]}")

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dim() < 1 or x.shape[-1] != self.normalized_shape[0]:
            raise ValueError(f"LayerNorm: expected [..., {self.normalized_shape[0]}], got {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)
