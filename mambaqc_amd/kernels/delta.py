"""The gated delta rule: a linear recurrence whose state is a matrix for each head, which a token first
reads at its key and then corrects there.

    p_t = exp(log_decay_t) S_{t-1},  r_t = v_t - p_t^T k_t,  S_t = p_t + beta_t k_t r_t^T,  o_t = scale S_t^T q_t

Beside gated_scan, whose state is one number a channel; the reference's block has neither (its state is a
quaternion for each channel and state index, models/quaternion_mamba2_block.py:206-228).
"""
from __future__ import annotations

import torch

from .. import _native as nat

MAX_KEY = 128  # elements of a key


def _check(name, q, k, v, log_decay, beta, h0, reset=None):
    if q.dim() != 4 or v.dim() != 4 or k.shape != q.shape or q.shape[:2] != v.shape[:2]:
        raise ValueError(f"{name}: q and k are [batch, seq_len, k_heads, k_dim] and v [batch, seq_len, "
                         f"v_heads, v_dim], got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    b, t, hv, dv = v.shape
    hk, dk = q.shape[2:]
    if min(hk, hv, dk, dv) < 1 or hv % hk:
        raise ValueError(f"{name}: {hv} value heads of {dv} are not a multiple of {hk} key heads of {dk}")
    if dk > MAX_KEY:
        raise ValueError(f"{name}: keys have at most {MAX_KEY} elements, got {dk}")
    for what, g in (("log_decay", log_decay), ("beta", beta)):
        if tuple(g.shape) != (b, t, hv):
            raise ValueError(f"{name}: {what} must be [{b}, {t}, {hv}], got {tuple(g.shape)}")
    if h0 is not None and tuple(h0.shape) != (b, hv, dk, dv):
        raise ValueError(f"{name}: the state must be [{b}, {hv}, {dk}, {dv}], got {tuple(h0.shape)}")
    if reset is not None and (tuple(reset.shape) != (b, t) or reset.dtype != torch.bool):
        raise ValueError(f"{name}: reset must be bool [{b}, {t}], got {reset.dtype} "
                         f"{tuple(reset.shape)}")


def _dtype(q, k, v) -> torch.dtype:
    return torch.promote_types(torch.promote_types(q.dtype, k.dtype), v.dtype)


def _saved(q, v):
    """Shapes of what a training forward stores: the chunks' states and residuals."""
    lib = nat.load()
    b, t, hv, dv = v.shape
    chunk = int(lib.mqc_gated_delta_chunk())
    width = int(lib.mqc_gated_delta_value_width(dv))
    lead = (b, hv, (t + chunk - 1) // chunk)
    return (*lead, int(lib.mqc_gated_delta_key_width(q.shape[3])), width), (*lead, chunk, width)


def _operands(name, q, k, v, log_decay, beta, reset=None, h0=None, scale=None):
    """The operands as the kernels read them; h0 is only looked at."""
    _check(name, q, k, v, log_decay, beta, h0, reset)
    return nat.host().Delta(name, q, k, v, log_decay, beta, reset, h0, scale)


def gated_delta(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                beta: torch.Tensor, h0: torch.Tensor | None = None,
                reset: torch.Tensor | None = None, scale: float | None = None,
                return_state: bool = False):
    """o [batch, seq_len, v_heads, v_dim] of the gated delta rule over q and k [batch, seq_len, k_heads,
    k_dim] and v [batch, seq_len, v_heads, v_dim] (in their promoted dtype; views whose last axis is dense,
    such as parts of a projection's output, are read in place), log_decay (at most 0) and beta [batch,
    seq_len, v_heads]. With return_state also the last state, fp32 [batch, v_heads, k_dim, v_dim].

    v_heads is a multiple of k_heads: consecutive value heads share a key head. k_dim is at most 128; keys
    are taken as they are (their layers make them of length one). h0: the state before the first token
    (None: zeros). reset: bool [batch, seq_len], true at the first token of a packed document: nothing
    from before it is seen, NaN included (in gradients, NaN and infinities reach up to 63 tokens to either
    side, over resets too). scale: of o, k_dim^-0.5 if None. States are fp32. A NaN or an infinity at a
    token may reach outputs of its own document up to 63 tokens before it. Differentiable in every tensor
    argument when autograd is recording (in reverse; forward mode is refused)."""
    if nat.compiling():
        _check("gated_delta", q, k, v, log_decay, beta, h0, reset)
        train = torch.is_grad_enabled() and any(x is not None and x.requires_grad
                                                for x in (q, k, v, log_decay, beta, h0))
        op = torch.ops.mambaqc.gated_delta_train if train else torch.ops.mambaqc.gated_delta
        o, h_last = op(q, k, v, log_decay, beta, h0, reset, scale)[:2]
    else:
        got = nat.host().gated_delta(q, k, v, log_decay, beta, h0, reset, scale)
        if got is None:  # say what is wrong
            _check("gated_delta", q, k, v, log_decay, beta, h0, reset)
        o, h_last = got
    return (o, h_last) if return_state else o


def gated_delta_step_(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                      beta: torch.Tensor, h: torch.Tensor, scale: float | None = None) -> torch.Tensor:
    """One token of the gated delta rule for each sequence: arguments as gated_delta's with seq_len 1 and
    the state h, contiguous fp32 [batch, v_heads, k_dim, v_dim], updated in place. Returns o [batch, 1,
    v_heads, v_dim]. No autograd (the decode step)."""
    o = nat.host().gated_delta_step(q, k, v, log_decay, beta, h, scale)
    if o is None:  # say what is wrong
        _check("gated_delta_step_", q, k, v, log_decay, beta, h)
        if v.shape[1] != 1:
            raise ValueError(f"gated_delta_step_: one token a sequence, got {v.shape[1]}")
        raise ValueError(f"gated_delta_step_: h must be contiguous float32, got {h.dtype}")
    return o
