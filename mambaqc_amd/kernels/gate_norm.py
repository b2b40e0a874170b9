"""What stands between two blocks of a stack: gate, norm after the block, scaled residual, norm before
the next block, in one pass over each row.

    v = sigmoid(z) y,  r = v / rms(v) post_weight,  out = x + scale r,  n = out / rms(out) pre_weight

with rms(u) = sqrt(mean u^2 + eps) over the last axis. The block's own output step is the first half
without the norms (the reference's models/quaternion_mamba2_block.py:157-161, `mambaqc_amd.out_gate`);
its LM normalises before the head only (models/quaternion_mamba2.py:158-163).
"""
from __future__ import annotations

import torch

from .. import _native as nat


def _check(x, y, z, post_weight, scale, pre_weight):
    if x.dim() < 1 or y.shape != x.shape:
        raise ValueError(f"gate_norm_residual: x and y are of one shape, got {tuple(x.shape)}, "
                         f"{tuple(y.shape)}")
    if z is not None and z.shape != x.shape:
        raise ValueError(f"gate_norm_residual: z must be {tuple(x.shape)}, got {tuple(z.shape)}")
    d = x.shape[-1]
    for name, w in (("post_weight", post_weight), ("scale", scale), ("pre_weight", pre_weight)):
        if w is not None and tuple(w.shape) != (d,):
            raise ValueError(f"gate_norm_residual: {name} must be [{d}], got {tuple(w.shape)}")


def _dtype(x, y, z) -> torch.dtype:
    t = torch.promote_types(x.dtype, y.dtype)
    return t if z is None else torch.promote_types(t, z.dtype)


def _z_rows(z: torch.Tensor, dtype: torch.dtype):
    """(z, elements between rows) in dtype, read in place where its rows are evenly spaced and its
    last axis is dense (the gate half of a projection's output)."""
    return nat.host().spaced_rows(z, dtype)


def _operands(x, y, z, post_weight, scale, pre_weight):
    """The operands as the kernels read them, weights in fp32."""
    _check(x, y, z, post_weight, scale, pre_weight)
    return nat.host().GateNorm(x, y, z, post_weight, scale, pre_weight, nat.param_f32)


def gate_norm_residual(x: torch.Tensor, y: torch.Tensor, z: torch.Tensor | None = None, *,
                       scale: torch.Tensor, pre_weight: torch.Tensor,
                       post_weight: torch.Tensor | None = None, eps: float = 1e-6):
    """(out, n) for x, y and z of one shape [..., d] (in their promoted dtype; z may be a strided view
    whose last axis is dense, read in place) and weights [d]:

        out = x + scale * rms_norm(sigmoid(z) * y) * post_weight,  n = rms_norm(out) * pre_weight

    without z the gate is 1, without post_weight y is not normalised. x is the residual stream, y a
    block's output, out the stream after it and n the next block's input. Norms and sums are fp32,
    and n comes from out before its rounding. d is at most 8192. Differentiable in every tensor
    argument when autograd is recording (in reverse; forward mode is refused)."""
    if nat.compiling():
        _check(x, y, z, post_weight, scale, pre_weight)
        return torch.ops.mambaqc.gate_norm_residual(x, y, z, post_weight, scale, pre_weight, eps)[:2]
    got = nat.host().gate_norm(x, y, z, post_weight, scale, pre_weight, eps, nat.param_f32)
    if got is None:  # say what is wrong
        _check(x, y, z, post_weight, scale, pre_weight)
    return got
