"""The gated scan: a linear recurrence with a real state for each channel, the block's SSM with a
real pole in place of the quaternion one and without its B and C.

    D_t = softplus(dt_raw_t),  a_t = exp(-D_t exp(log_rate)),  s_t = sigmoid(g_raw_t) x_t
    h_t = a_t h_{t-1} + (1 - a_t) s_t

dt_raw, g_raw and x are what ssm_front takes; log_rate is [width]. The reference's Lite block is the
nearest it has (a real state walked by a Python loop over time,
models/quaternion_mamba2_lite_block.py:143-154).
"""
from __future__ import annotations

import torch

from .. import _native as nat


def _rows(t: torch.Tensor, dtype: torch.dtype):
    """(t, elements between tokens) in dtype, read in place where its tokens are evenly spaced and
    its last axis is dense."""
    b, n, d = t.shape
    t = t.detach().to(dtype)
    if (d > 1 and t.stride(2) != 1) or (b > 1 and n > 1 and t.stride(0) != n * t.stride(1)) or (
            b * n > 1 and (t.stride(1) if n > 1 else t.stride(0)) < d):
        t = t.contiguous()
    return t, d if b * n <= 1 else t.stride(1) if n > 1 else t.stride(0)


def _check(name, dt_raw, g_raw, x, log_rate, h0, reset=None):
    if x.dim() != 3 or not dt_raw.shape == g_raw.shape == x.shape:
        raise ValueError(f"{name}: dt_raw, g_raw and x are [batch, seq_len, width] of one shape, got "
                         f"{tuple(dt_raw.shape)}, {tuple(g_raw.shape)}, {tuple(x.shape)}")
    b, t, d = x.shape
    if tuple(log_rate.shape) != (d,):
        raise ValueError(f"{name}: log_rate must be [{d}], got {tuple(log_rate.shape)}")
    if h0 is not None and tuple(h0.shape) != (b, d):
        raise ValueError(f"{name}: the state must be [{b}, {d}], got {tuple(h0.shape)}")
    if reset is not None and (tuple(reset.shape) != (b, t) or reset.dtype != torch.bool):
        raise ValueError(f"{name}: reset must be bool [{b}, {t}], got {reset.dtype} "
                         f"{tuple(reset.shape)}")


def _scan_dtype(dt_raw, g_raw, x) -> torch.dtype:
    return torch.promote_types(torch.promote_types(dt_raw.dtype, g_raw.dtype), x.dtype)


def scan_chunk() -> int:
    """Steps between the states that a training forward stores."""
    return int(nat.load().mqc_gated_scan_chunk())


def _scan_forward(dt_raw, g_raw, x, log_rate, h0, reset, train):
    """(y, h_last, carries or None, the operands as the kernels read them)."""
    nat.require_device("gated_scan", x, dt_raw, g_raw, log_rate,
                       *(v for v in (h0, reset) if v is not None))
    b, t, d = x.shape
    ct = _scan_dtype(dt_raw, g_raw, x)
    (dt, dts), (g, gs), (xv, xs) = (_rows(v, ct) for v in (dt_raw, g_raw, x))
    lam = nat.param_f32(log_rate)
    h0 = None if h0 is None else h0.detach().float().contiguous()
    reset = None if reset is None else reset.detach().contiguous()
    y = torch.empty(b, t, d, device=x.device, dtype=ct)
    h_last = torch.empty(b, d, device=x.device, dtype=torch.float32)
    lib = nat.load()
    carries = None
    if train:
        every = scan_chunk()
        carries = torch.empty(b, (t + every - 1) // every, d, device=x.device,
                              dtype=torch.float32)
    nbytes = lib.mqc_gated_scan_workspace_bytes(b, t, d)
    ws = torch.empty(nbytes, device=x.device, dtype=torch.uint8)
    nat.call("mqc_gated_scan_fwd", xv, dt.data_ptr(), dts, g.data_ptr(), gs, xv.data_ptr(), xs,
             lam.data_ptr(), nat.ptr(h0), nat.ptr(reset), y.data_ptr(), h_last.data_ptr(),
             nat.ptr(carries), b, t, d, nat.dtype_code(xv), ws.data_ptr(), nbytes,
             nat.stream_of(xv))
    return y, h_last, carries, (dt, g, xv, lam, reset)


def _scan_backward(operands, carries, dy, dh_last, want_dh0):
    """(ddt, dg, dx in the operands' dtype, dlog_rate, dh0 or None in fp32)."""
    dt_raw, g_raw, x, lam, reset = operands
    b, t, d = x.shape
    if x.numel() == 0:
        grads = [torch.empty_like(x, memory_format=torch.contiguous_format) for _ in range(3)]
        dh0 = None
        if want_dh0:
            dh0 = (torch.zeros(b, d, device=x.device) if dh_last is None
                   else dh_last.float().clone())
        return (*grads, torch.zeros_like(lam), dh0)
    (dt, dts), (g, gs), (xv, xs) = (_rows(v, x.dtype) for v in (dt_raw, g_raw, x))
    dy = (torch.zeros(b, t, d, device=x.device, dtype=x.dtype) if dy is None
          else dy.to(x.dtype).contiguous())
    dh_last = None if dh_last is None else dh_last.float().contiguous()
    ddt, dg, dx = (torch.empty(b, t, d, device=x.device, dtype=x.dtype) for _ in range(3))
    drate = torch.empty(d, device=x.device, dtype=torch.float32)
    dh0 = torch.empty(b, d, device=x.device, dtype=torch.float32) if want_dh0 else None
    nbytes = nat.load().mqc_gated_scan_workspace_bytes(b, t, d)
    ws = torch.empty(nbytes, device=x.device, dtype=torch.uint8)
    nat.call("mqc_gated_scan_bwd", xv, dt.data_ptr(), dts, g.data_ptr(), gs, xv.data_ptr(), xs,
             lam.data_ptr(), nat.ptr(reset), carries.data_ptr(), dy.data_ptr(), nat.ptr(dh_last),
             ddt.data_ptr(), dg.data_ptr(), dx.data_ptr(), drate.data_ptr(), nat.ptr(dh0), b, t, d,
             nat.dtype_code(xv), ws.data_ptr(), nbytes, nat.stream_of(xv))
    return ddt, dg, dx, drate, dh0


class _GatedScan(torch.autograd.Function):
    """The scan with HIP forward (storing the chunks' entry states) and backward."""

    @staticmethod
    def forward(ctx, dt_raw, g_raw, x, log_rate, h0, reset):
        y, h_last, carries, ops = _scan_forward(dt_raw, g_raw, x, log_rate, h0, reset, True)
        ctx.save_for_backward(*ops, carries)
        ctx.set_materialize_grads(False)
        ctx.meta = (dt_raw.dtype, g_raw.dtype, x.dtype, log_rate.dtype,
                    None if h0 is None else h0.dtype)
        return y, h_last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh_last):
        *ops, carries = ctx.saved_tensors
        t_dt, t_g, t_x, t_rate, t_h0 = ctx.meta
        ddt, dg, dx, drate, dh0 = _scan_backward(ops, carries, dy, dh_last,
                                                 t_h0 is not None and ctx.needs_input_grad[4])
        return (ddt.to(t_dt), dg.to(t_g), dx.to(t_x), drate.to(t_rate),
                None if dh0 is None else dh0.to(t_h0), None)


def gated_scan(dt_raw: torch.Tensor, g_raw: torch.Tensor, x: torch.Tensor, log_rate: torch.Tensor,
               h0: torch.Tensor | None = None, reset: torch.Tensor | None = None,
               return_state: bool = False):
    """y [batch, seq_len, width] of the gated scan over dt_raw, g_raw and x (one shape, in their
    promoted dtype; views with evenly spaced tokens, such as parts of a projection's output, are
    read in place), log_rate [width]. With return_state also the last state, fp32 [batch, width].

    h0: the state before the first token (None: zeros). reset: bool [batch, seq_len], true at the
    first token of a packed document: nothing from before it is seen, NaN included. States are
    fp32. Differentiable in every tensor argument when autograd is recording."""
    _check("gated_scan", dt_raw, g_raw, x, log_rate, h0, reset)
    train = torch.is_grad_enabled() and any(v is not None and v.requires_grad
                                            for v in (dt_raw, g_raw, x, log_rate, h0))
    if nat.compiling():
        op = torch.ops.mambaqc.gated_scan_train if train else torch.ops.mambaqc.gated_scan
        y, h_last = op(dt_raw, g_raw, x, log_rate, h0, reset)[:2]
    elif train:
        y, h_last = _GatedScan.apply(dt_raw, g_raw, x, log_rate, h0, reset)
    else:
        y, h_last, _, _ = _scan_forward(dt_raw, g_raw, x, log_rate, h0, reset, False)
    return (y, h_last) if return_state else y


def gated_scan_step_(dt_raw: torch.Tensor, g_raw: torch.Tensor, x: torch.Tensor,
                     log_rate: torch.Tensor, h: torch.Tensor) -> torch.Tensor:
    """One token of the gated scan for each sequence: dt_raw, g_raw, x [batch, 1, width] and the
    state h, contiguous fp32 [batch, width], updated in place. Returns y [batch, 1, width]. No
    autograd (the decode step)."""
    _check("gated_scan_step_", dt_raw, g_raw, x, log_rate, h)
    b, t, d = x.shape
    if t != 1:
        raise ValueError(f"gated_scan_step_: one token a sequence, got {t}")
    if h.dtype != torch.float32 or not h.is_contiguous():
        raise ValueError(f"gated_scan_step_: h must be contiguous float32, got {h.dtype}")
    nat.require_device("gated_scan_step_", x, dt_raw, g_raw, log_rate, h)
    ct = _scan_dtype(dt_raw, g_raw, x)
    (dt, dts), (g, gs), (xv, xs) = (_rows(v, ct) for v in (dt_raw, g_raw, x))
    y = torch.empty(b, 1, d, device=x.device, dtype=ct)
    nat.call("mqc_gated_scan_step", xv, dt.data_ptr(), dts, g.data_ptr(), gs, xv.data_ptr(), xs,
             nat.param_f32(log_rate).data_ptr(), h.data_ptr(), y.data_ptr(), b, d,
             nat.dtype_code(xv), nat.stream_of(xv))
    return y
