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
    """(t [b, n, d], elements between tokens) in dtype, read in place where its tokens are evenly
    spaced and its last axis is dense."""
    return nat.host().token_rows(t, dtype)


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


def _operands(name, dt_raw, g_raw, x, log_rate, reset=None, h0=None):
    """The operands as the kernels read them, log_rate in fp32; h0 is only looked at."""
    _check(name, dt_raw, g_raw, x, log_rate, h0, reset)
    return nat.host().Scan(name, dt_raw, g_raw, x, log_rate, reset, h0, nat.param_f32)


def _state(h0):
    return None if h0 is None else h0.detach().float().contiguous()


def gated_scan(dt_raw: torch.Tensor, g_raw: torch.Tensor, x: torch.Tensor, log_rate: torch.Tensor,
               h0: torch.Tensor | None = None, reset: torch.Tensor | None = None,
               return_state: bool = False):
    """y [batch, seq_len, width] of the gated scan over dt_raw, g_raw and x (one shape, in their
    promoted dtype; views with evenly spaced tokens, such as parts of a projection's output, are
    read in place), log_rate [width]. With return_state also the last state, fp32 [batch, width].

    h0: the state before the first token (None: zeros). reset: bool [batch, seq_len], true at the
    first token of a packed document: nothing from before it is seen, NaN included. States are
    fp32. Differentiable in every tensor argument when autograd is recording (in reverse; forward mode
    is refused)."""
    if nat.compiling():
        _check("gated_scan", dt_raw, g_raw, x, log_rate, h0, reset)
        train = torch.is_grad_enabled() and any(v is not None and v.requires_grad
                                                for v in (dt_raw, g_raw, x, log_rate, h0))
        op = torch.ops.mambaqc.gated_scan_train if train else torch.ops.mambaqc.gated_scan
        y, h_last = op(dt_raw, g_raw, x, log_rate, h0, reset)[:2]
    else:
        got = nat.host().gated_scan(dt_raw, g_raw, x, log_rate, h0, reset, nat.param_f32)
        if got is None:  # say what is wrong
            _check("gated_scan", dt_raw, g_raw, x, log_rate, h0, reset)
        y, h_last = got
    return (y, h_last) if return_state else y


def gated_scan_step_(dt_raw: torch.Tensor, g_raw: torch.Tensor, x: torch.Tensor,
                     log_rate: torch.Tensor, h: torch.Tensor) -> torch.Tensor:
    """One token of the gated scan for each sequence: dt_raw, g_raw, x [batch, 1, width] and the
    state h, contiguous fp32 [batch, width], updated in place. Returns y [batch, 1, width]. No
    autograd (the decode step)."""
    y = nat.host().gated_scan_step(dt_raw, g_raw, x, log_rate, h, nat.param_f32)
    if y is None:  # say what is wrong
        _check("gated_scan_step_", dt_raw, g_raw, x, log_rate, h)
        if x.shape[1] != 1:
            raise ValueError(f"gated_scan_step_: one token a sequence, got {x.shape[1]}")
        raise ValueError(f"gated_scan_step_: h must be contiguous float32, got {h.dtype}")
    return y
