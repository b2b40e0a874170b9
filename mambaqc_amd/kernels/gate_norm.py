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


def _z_rows(z, dtype):
    """(z, elements between rows) in dtype, read in place where its rows are evenly spaced and its
    last axis is dense (the gate half of a projection's output)."""
    d = z.shape[-1]
    z = z.detach().to(dtype)
    row, want = None, None
    for n, s in zip(reversed(z.shape[:-1]), reversed(z.stride()[:-1])):
        if n == 1:
            continue
        if row is None:
            row = s
        elif s != want:
            row = 0
            break
        want = s * n
    if row is None:
        row = d
    if (d > 1 and z.stride(-1) != 1) or row < d:
        z, row = z.contiguous(), d
    return z, row


def _operands(x, y, z, post_weight, scale, pre_weight):
    """The operands as the kernels read them: (x, y, z, z's row, weights in fp32)."""
    ct = _dtype(x, y, z)
    x, y = x.detach().to(ct).contiguous(), y.detach().to(ct).contiguous()
    z, z_row = (None, 0) if z is None else _z_rows(z, ct)
    post = None if post_weight is None else nat.param_f32(post_weight)
    return x, y, z, z_row, post, nat.param_f32(scale), nat.param_f32(pre_weight)


def _forward(operands, eps, train):
    """(out, n, the rows' inverse norms or None)."""
    x, y, z, z_row, post, scale, pre = operands
    d = x.shape[-1]
    out, n = torch.empty_like(x), torch.empty_like(x)
    rows = x.numel() // d if d else 0
    stats = torch.empty(rows, 2, device=x.device, dtype=torch.float32) if train else None
    if rows:
        nat.call("mqc_gate_norm_fwd", x, x.data_ptr(), y.data_ptr(), nat.ptr(z), z_row,
                 nat.ptr(post), scale.data_ptr(), pre.data_ptr(), out.data_ptr(), n.data_ptr(),
                 nat.ptr(stats), rows, d, float(eps), nat.dtype_code(x), nat.stream_of(x))
    return out, n, stats


def _backward(operands, stats, dout, dn):
    """(dx, dy, dz or None in the operands' dtype, dpost or None, dscale, dpre in fp32); dout or dn
    None for zeros."""
    x, y, z, z_row, post, scale, pre = operands
    d = x.shape[-1]
    rows = x.numel() // d if d else 0
    dx, dy = torch.empty_like(x), torch.empty_like(x)
    dz = None if z is None else torch.empty_like(x)
    dscale, dpre = torch.empty_like(scale), torch.empty_like(pre)
    dpost = None if post is None else torch.empty_like(post)
    if not rows:
        return dx, dy, dz, None if dpost is None else dpost.zero_(), dscale.zero_(), dpre.zero_()
    dout, dn = (None if v is None else v.to(x.dtype).contiguous() for v in (dout, dn))
    nbytes = nat.load().mqc_gate_norm_workspace_bytes(rows, d)
    ws = torch.empty(nbytes, device=x.device, dtype=torch.uint8)
    nat.call("mqc_gate_norm_bwd", x, x.data_ptr(), y.data_ptr(), nat.ptr(z), z_row, nat.ptr(post),
             scale.data_ptr(), pre.data_ptr(), stats.data_ptr(), nat.ptr(dout), nat.ptr(dn),
             dx.data_ptr(), dy.data_ptr(), nat.ptr(dz), nat.ptr(dpost), dscale.data_ptr(),
             dpre.data_ptr(), rows, d, nat.dtype_code(x), ws.data_ptr(), nbytes, nat.stream_of(x))
    return dx, dy, dz, dpost, dscale, dpre


class _GateNormResidual(torch.autograd.Function):
    """HIP forward (storing the rows' inverse norms) and backward."""

    @staticmethod
    def forward(ctx, x, y, z, post_weight, scale, pre_weight, eps):
        ops = _operands(x, y, z, post_weight, scale, pre_weight)
        out, n, stats = _forward(ops, eps, True)
        ctx.save_for_backward(*ops[:3], *ops[4:], stats)
        ctx.set_materialize_grads(False)
        ctx.z_row = ops[3]
        ctx.types = [None if v is None else v.dtype for v in (x, y, z, post_weight, scale, pre_weight)]
        return out, n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dn):
        *ops, stats = ctx.saved_tensors
        grads = _backward((*ops[:3], ctx.z_row, *ops[3:]), stats, dout, dn)
        return (*(None if g is None else g.to(t) for g, t in zip(grads, ctx.types)), None)


def gate_norm_residual(x: torch.Tensor, y: torch.Tensor, z: torch.Tensor | None = None, *,
                       scale: torch.Tensor, pre_weight: torch.Tensor,
                       post_weight: torch.Tensor | None = None, eps: float = 1e-6):
    """(out, n) for x, y and z of one shape [..., d] (in their promoted dtype; z may be a strided view
    whose last axis is dense, read in place) and weights [d]:

        out = x + scale * rms_norm(sigmoid(z) * y) * post_weight,  n = rms_norm(out) * pre_weight

    without z the gate is 1, without post_weight y is not normalised. x is the residual stream, y a
    block's output, out the stream after it and n the next block's input. Norms and sums are fp32,
    and n comes from out before its rounding. d is at most 8192. Differentiable in every tensor
    argument when autograd is recording."""
    _check(x, y, z, post_weight, scale, pre_weight)
    tensors = [v for v in (x, y, z, post_weight, scale, pre_weight) if v is not None]
    train = torch.is_grad_enabled() and any(v.requires_grad for v in tensors)
    if nat.compiling():
        return torch.ops.mambaqc.gate_norm_residual(x, y, z, post_weight, scale, pre_weight, eps)[:2]
    nat.require_device("gate_norm_residual", *tensors)
    if train:
        return _GateNormResidual.apply(x, y, z, post_weight, scale, pre_weight, eps)
    return _forward(_operands(x, y, z, post_weight, scale, pre_weight), eps, False)[:2]
