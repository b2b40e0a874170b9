"""AdamW and Muon on the GPU.

AdamW: one launch for 88 tensors of a dtype (60 with 8-bit states), states in 32 or in 8 bits, the
gradients' norm and its clipping on the device.

    p <- p (1 - lr weight_decay) - lr m^ / (sqrt(v^) + eps),  m^ = m / (1 - beta1^t),  v^ = v / (1 - beta2^t)

computed in fp32 from p and its gradient in their own dtype (fp32, bf16 or fp16), and rounded to p's
dtype once. `AdamW` is the torch.optim.Optimizer (the reference's trainer uses torch's, train.py:182-206:
clip to 1.0, then the step); `adamw_step_`, `adamw8_step_` and `grad_norm` are the operators under it.

8-bit states hold m and sqrt(v) as torch.float8_e4m3fn with a power-of-two scale for each 256 elements
of a tensor: 2.03 bytes a parameter instead of 8 (a 14.66 B parameter model: 30 GB instead of 117).
Their rounding keeps the means of m and of v (csrc/adamw.hip); it needs a seed, and the same seed and
step give the same bits.

Muon, for matrices: momentum, the nearest orthogonal matrix by Newton's and Schulz's iteration, the step.

    m <- mu m + (1 - mu) g,  u = mu m + (1 - mu) g (nesterov) or m,  X = u / max(|u|_F, eps)
    X <- a X + (b A + c A^2) X with A = X X^T, `steps` times
    p <- p (1 - lr weight_decay) - lr max(1, rows / cols)^1/2 X

`Muon` is the optimizer, `muon_step_` and `orthogonalize` are the operators under it (csrc/ortho.hip). All
matrices of a type go through the same launches, up to 64 of 16 shapes at a time.
"""
from __future__ import annotations

import array
import bisect
import collections
import itertools
import math

import torch

from . import _native as nat

STATE_BLOCK = 256  # elements that share a scale


def state_blocks(numel: int) -> int:
    """Scales of an 8-bit state of numel elements."""
    return -(-numel // STATE_BLOCK)


def _check_lengths(name, *lists):
    if not all(len(s) == len(lists[0]) for s in lists):
        raise ValueError(f"{name}: lists of different lengths {[len(s) for s in lists]}")


def _check_tensors(name, params, grads, *states):
    """params and grads of one device, dtypes and shapes that match, all dense."""
    for p, g in zip(params, grads):
        if p.shape != g.shape or p.dtype != g.dtype:
            raise ValueError(f"{name}: a gradient is {g.dtype} {tuple(g.shape)}, its parameter "
                             f"{p.dtype} {tuple(p.shape)}")
        if g.layout != torch.strided or not p.is_contiguous() or not g.is_contiguous():
            raise ValueError(f"{name}: parameters and gradients must be contiguous")
        nat.dtype_code(p)
    flat = list(itertools.chain(params, grads, *states))
    if flat:
        nat.require_device(name, *flat)


def _check_state(name, what, params, states, dtype, count=None):
    for p, s in zip(params, states):
        numel = p.numel() if count is None else count(p.numel())
        if s.dtype != dtype or s.numel() != numel or not s.is_contiguous():
            raise ValueError(f"{name}: {what} must be contiguous {dtype} of {numel} elements, got "
                             f"{s.dtype} of {s.numel()}")


def _scalars(step, lr, betas, eps, weight_decay):
    if step < 1:
        raise ValueError(f"adamw: steps count from 1, got {step}")
    (b1, b2), lr = betas, float(lr)
    return (1 - lr * weight_decay, lr / (1 - b1 ** step), 1 / math.sqrt(1 - b2 ** step), b1, 1 - b1,
            b2, 1 - b2, eps)


def _tables(name, params, grads, states, scales, seeds):
    """The rows that mqc_adamw_step or mqc_adamw8_step reads, and mqc_grad_norm's."""
    got = nat.host().adam_rows((params, grads, *states, *scales), STATE_BLOCK, seeds)
    if got is None:  # say what is wrong
        eight = len(scales) > 0
        for s in states:
            _check_state(name, "states", params, s, torch.float8_e4m3fn if eight else torch.float32)
        for s in scales:
            _check_state(name, "scales", params, s, torch.float32, state_blocks)
        _check_tensors(name, params, grads, *states, *scales)
        spans = sorted((p.data_ptr(), p.data_ptr() + p.nbytes) for p in params if p.numel())
        if any(b[0] < a[1] for a, b in zip(spans, spans[1:])):
            raise ValueError(f"{name}: a parameter is there twice, or two of them share memory")
        raise ValueError(f"{name}: tensors that the kernels do not take")
    return got


def _norm_and_clip(rows: bytes, max_norm, like):
    """(norm, clip) as fp32 scalars on the gradients' device, from mqc_grad_norm's rows."""
    count = len(rows) // 24
    nbytes = nat.load().mqc_grad_norm_workspace_bytes(rows, count)
    if nbytes < 0:
        nat.check(nbytes, "mqc_grad_norm")
    out = torch.empty(2, device=like.device, dtype=torch.float32)
    ws = torch.empty(nbytes, device=like.device, dtype=torch.uint8)
    at = out.data_ptr()
    nat.call("mqc_grad_norm", out, rows, count, float(max_norm), at, at + 4, ws.data_ptr(),
             nbytes, nat.stream_of(out))
    return out[0], out[1]


def grad_norm(grads: list[torch.Tensor]) -> torch.Tensor:
    """The 2-norm of all elements of the tensors together (fp32 scalar on their device; summed in 64
    bits, in a fixed order)."""
    if not grads:
        raise ValueError("grad_norm: no tensors")
    _check_tensors("grad_norm", grads, grads)
    rows = array.array("q", [v for g in grads for v in (g.data_ptr(), g.numel(), nat.dtype_code(g))])
    return _norm_and_clip(rows.tobytes(), math.inf, grads[0])[0]


def adamw_step_(params, grads, exp_avgs, exp_avg_sqs, *, step: int, lr: float = 1e-3,
                betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                max_norm: float | None = None) -> torch.Tensor | None:
    """One AdamW step in place over lists of tensors: contiguous parameters and gradients of one
    dtype each (fp32, bf16 or fp16), no two parameters in the same memory, fp32 states. step counts
    from 1. With max_norm the gradients are scaled by min(1, max_norm / (norm + 1e-6)) as they are
    read (they stay as they are), norm over all of them, which is returned (fp32 scalar on the
    device)."""
    params, grads = list(params), list(grads)
    how = _scalars(step, lr, betas, eps, weight_decay)
    states = (exp_avgs, exp_avg_sqs)
    _check_lengths("adamw_step_", params, grads, *states)
    if not params:
        return None
    rows, norm_rows = _tables("adamw_step_", params, grads, states, (), ())
    norm, clip = (None, None) if max_norm is None else _norm_and_clip(norm_rows, max_norm, params[0])
    _launch32(rows, params, states, how, clip)
    return norm


def _launch32(rows, params, states, how, clip):
    nat.call("mqc_adamw_step", params[0], rows, len(params), *how, nat.ptr(clip),
             nat.stream_of(params[0]))
    # The kernels write through pointers: tell autograd (and whatever keeps copies of parameters by
    # their version, as param_f32 does) that these tensors changed.
    nat.host().changed((params, *states))


def adamw8_step_(params, grads, exp_avgs, exp_avg_scales, root_avg_sqs, root_avg_sq_scales, *,
                 step: int, seed: int = 0, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, max_norm: float | None = None) -> torch.Tensor | None:
    """adamw_step_ with states in 8 bits: exp_avgs and root_avg_sqs (sqrt(v)) torch.float8_e4m3fn
    tensors of the parameters' sizes, their scales fp32 of state_blocks(numel) elements. What a state
    stands for is its value times its block's scale. Tensor i of the lists rounds by seed + i."""
    params, grads = list(params), list(grads)
    how = _scalars(step, lr, betas, eps, weight_decay)
    states, scales = (exp_avgs, root_avg_sqs), (exp_avg_scales, root_avg_sq_scales)
    _check_lengths("adamw8_step_", params, grads, *states, *scales)
    if not params:
        return None
    rows, norm_rows = _tables("adamw8_step_", params, grads, states, scales,
                              [(seed + i) & 0xFFFFFFFF for i in range(len(params))])
    norm, clip = (None, None) if max_norm is None else _norm_and_clip(norm_rows, max_norm, params[0])
    _launch8(rows, params, (*states, *scales), how, clip, step)
    return norm


def _launch8(rows, params, states, how, clip, step):
    nat.call("mqc_adamw8_step", params[0], rows, len(params), *how, nat.ptr(clip),
             step & 0xFFFFFFFF, nat.stream_of(params[0]))
    nat.host().changed((params, *states))


def _viewed(state, from_dtype, to_dtype):
    """A parameter's state with its tensors of one 8-bit type viewed as the other."""
    return {k: v.view(to_dtype) if isinstance(v, torch.Tensor) and v.dtype == from_dtype else v
            for k, v in state.items()}


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay over the kernels of this module.

    state_bits: 32, or 8 for e4m3 states of the parameters with at least min_8bit_size elements
    (smaller ones keep 32: they are no memory, and norms and gains are the ones that matter).
    max_norm: the gradients' norm, over all groups together, is clipped to it as they are read;
    `grad_norm` holds the last step's norm (a device scalar, not clipped). seed: of the 8-bit states'
    rounding. Steps and learning rates are the host's: a step is not captured into a graph."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, state_bits: int = 32, min_8bit_size: int = 4096,
                 max_norm: float | None = None, seed: int = 0):
        if lr < 0 or eps < 0 or weight_decay < 0:
            raise ValueError(f"AdamW: lr {lr}, eps {eps} and weight_decay {weight_decay} are not "
                             "negative")
        if not all(0 <= b < 1 for b in betas):
            raise ValueError(f"AdamW: betas are in [0, 1), got {betas}")
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits is 8 or 32, got {state_bits}")
        super().__init__(params, {"lr": lr, "betas": tuple(betas), "eps": eps,
                                  "weight_decay": weight_decay, "state_bits": state_bits})
        self.min_8bit_size, self.max_norm, self.seed = min_8bit_size, max_norm, seed
        self.grad_norm = None

    def __getstate__(self):
        """What copies and pickles take along: torch's part, with 8-bit states as bytes (float8 tensors
        cannot be unpickled), and this class's own settings."""
        got = super().__getstate__()
        got |= {k: getattr(self, k) for k in ("min_8bit_size", "max_norm", "seed", "grad_norm")}
        got["state"] = collections.defaultdict(dict, {p: _viewed(s, torch.float8_e4m3fn, torch.uint8)
                                                      for p, s in self.state.items()})
        return got

    def __setstate__(self, state):
        super().__setstate__(state)
        for p, s in self.state.items():
            self.state[p] = _viewed(s, torch.uint8, torch.float8_e4m3fn)

    def _state_of(self, p, bits):
        s = self.state[p]
        if not s:
            s["step"] = 0
            if bits == 8 and p.numel() >= self.min_8bit_size:
                for k in ("exp_avg", "root_avg_sq"):
                    s[k] = torch.zeros(p.shape, device=p.device, dtype=torch.uint8).view(
                        torch.float8_e4m3fn)
                    s[k + "_scale"] = torch.ones(state_blocks(p.numel()), device=p.device,
                                                 dtype=torch.float32)
            else:
                s["exp_avg"] = torch.zeros(p.shape, device=p.device, dtype=torch.float32)
                s["exp_avg_sq"] = torch.zeros(p.shape, device=p.device, dtype=torch.float32)
        return s

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: a step counts on the host and is not captured into a graph")
        todo, place = {}, 0
        for index, group in enumerate(self.param_groups):
            for p in group["params"]:
                place += 1
                if p.grad is None:
                    continue
                if p.grad.layout != torch.strided:
                    raise ValueError("AdamW: sparse gradients are not supported")
                g = p.grad.detach().contiguous().resolve_neg()
                if g.dtype != p.dtype:
                    g = g.to(p.dtype)
                s = self._state_of(p, group["state_bits"])
                todo.setdefault((index, s["step"], "root_avg_sq" in s), []).append(
                    (p.detach(), g, s, (self.seed + place) & 0xFFFFFFFF))
        if not todo:
            return loss
        work = []
        for (index, step, eight), entries in todo.items():
            params, grads, states, seeds = zip(*entries)
            keys = ("exp_avg", "root_avg_sq") if eight else ("exp_avg", "exp_avg_sq")
            held = [[s[k] for s in states] for k in keys]
            scales = [[s[k + "_scale"] for s in states] for k in keys] if eight else []
            work.append((index, step, params, states, held + scales,
                         _tables("AdamW", params, grads, held, scales, seeds)))
        clip = None
        if self.max_norm is not None:
            nat.require_device("AdamW", *(w[2][0] for w in work))  # one norm, on one device
            self.grad_norm, clip = _norm_and_clip(b"".join(w[-1][1] for w in work), self.max_norm,
                                                  work[0][2][0])
        for index, step, params, states, held, (rows, _) in work:
            group = self.param_groups[index]
            how = _scalars(step + 1, group["lr"], group["betas"], group["eps"],
                           group["weight_decay"])
            if len(held) == 4:
                _launch8(rows, params, held, how, clip, step + 1)
            else:
                _launch32(rows, params, held, how, clip)
            for s in states:
                s["step"] = step + 1
        return loss

    def load_state_dict(self, state_dict):
        """torch's loading casts floating states to the parameter's dtype: the states' own are
        put back from what was saved."""
        super().load_state_dict(state_dict)
        ids = itertools.chain.from_iterable(g["params"] for g in state_dict["param_groups"])
        params = itertools.chain.from_iterable(g["params"] for g in self.param_groups)
        for i, p in zip(ids, params):
            saved = state_dict["state"].get(i)
            if saved is not None:
                self.state[p] = {k: v.detach().to(p.device, copy=True).contiguous()
                                 if isinstance(v, torch.Tensor) else v for k, v in saved.items()}


# --- orthogonalised updates of matrices ------------------------------------------------------------

COEFFICIENTS = (3.4445, -4.775, 2.0315)  # of Muon: a steep start, and an end between 0.7 and 1.2
_PAIRS = 16  # MQC_ORTHO_PAIRS


def _iteration(name, steps, coefficients, eps):
    if not 1 <= steps <= 100:
        raise ValueError(f"{name}: steps is 1 to 100, got {steps}")
    if len(coefficients) != 3:
        raise ValueError(f"{name}: three coefficients, got {coefficients}")
    if not eps >= 0:
        raise ValueError(f"{name}: eps is not negative, got {eps}")
    return (steps, *map(float, coefficients), eps)


def _code(x, fast_bf16):
    return nat.dtype_code(x) | (0 if fast_bf16 else _PAIRS)


def _workspace(nbytes, name, like):
    if nbytes < 0:
        nat.check(nbytes, name)
    return torch.empty(nbytes, device=like.device, dtype=torch.uint8)


@torch.no_grad()
def orthogonalize(x: torch.Tensor, steps: int = 5, coefficients=COEFFICIENTS,
                  eps: float = 1e-7, fast_bf16: bool = False) -> torch.Tensor:
    """x [..., rows, cols] (fp32, bf16 or fp16) after `steps` of Newton's and Schulz's iteration, in its
    dtype: each matrix over max(its 2-norm, eps), then X <- a X + (b A + c A^2) X with A = X X^T, which
    brings its singular values near 1. The coefficients have to keep the elements of X, of A and of b A + c A^2
    below 255 on the way (their singular values below it is enough): beyond, results are not finite.
    Everything is iterated at fp32's accuracy and rounded once. fast_bf16: bf16 matrices with a shorter side of
    256 or more with 11-bit operands instead, in half to two thirds of the time, off by 1e-3 (the type's own
    rounding: 1.7e-3). No autograd."""
    how = _iteration("orthogonalize", steps, coefficients, eps)
    if x.dim() < 2:
        raise ValueError(f"orthogonalize: x is [..., rows, cols], got {tuple(x.shape)}")
    dtype = _code(x, fast_bf16)
    nat.require_device("orthogonalize", x)
    x = x.detach().contiguous().resolve_neg()
    out = torch.empty_like(x)
    if x.numel() == 0:
        return out
    rows, cols = x.shape[-2:]
    batch = x.numel() // (rows * cols)
    nbytes = nat.load().mqc_orthogonalize_workspace_bytes(batch, rows, cols, dtype)
    ws = _workspace(nbytes, "mqc_orthogonalize", x)
    nat.call("mqc_orthogonalize", x, x.data_ptr(), out.data_ptr(), batch, rows, cols, *how, dtype,
             ws.data_ptr(), nbytes, nat.stream_of(x))
    return out


def _muon_rows(name, params, grads, momenta, fast_bf16=False):
    """The rows that mqc_muon_step reads."""
    _check_lengths(name, params, grads, momenta)
    for p in params:
        if p.dim() != 2:
            raise ValueError(f"{name}: parameters are matrices, got {tuple(p.shape)}")
    _check_state(name, "momenta", params, momenta, torch.float32)
    _check_tensors(name, params, grads, momenta)
    if any(t.is_neg() for t in itertools.chain(params, grads, momenta)):
        raise ValueError(f"{name}: tensors that the kernels do not take")
    written = [t for t in itertools.chain(params, momenta) if t.numel()]
    spans = sorted((t.data_ptr(), t.data_ptr() + t.nbytes) for t in written)
    if any(b[0] < a[1] for a, b in zip(spans, spans[1:])):
        raise ValueError(f"{name}: a parameter is there twice, or two of them share memory")
    starts = [start for start, _ in spans]
    for p, g in zip(params, grads):  # (momenta are written before gradients are read again)
        last = bisect.bisect_left(starts, g.data_ptr() + g.nbytes) - 1
        if g.numel() and g.data_ptr() != p.data_ptr() and last >= 0 and spans[last][1] > g.data_ptr():
            raise ValueError(f"{name}: a gradient shares memory with a momentum or another parameter")
    return [(p.data_ptr(), g.data_ptr(), m.data_ptr(), *p.shape, _code(p, fast_bf16))
            for p, g, m in zip(params, grads, momenta) if p.numel()]


@torch.no_grad()
def muon_step_(params, grads, momenta, *, lr: float = 1e-3, momentum: float = 0.95, nesterov: bool = True,
               weight_decay: float = 0.1, steps: int = 5, coefficients=COEFFICIENTS,
               eps: float = 1e-7, fast_bf16: bool = False) -> None:
    """One Muon step in place over lists of matrices: contiguous parameters and gradients of one dtype each
    (fp32, bf16 or fp16), fp32 momenta of their sizes, no two parameters in the same memory and no gradient in
    a momentum's. The iteration (and fast_bf16) is orthogonalize's."""
    params, grads, momenta = list(params), list(grads), list(momenta)
    how = _iteration("muon_step_", steps, coefficients, eps)
    rows = _muon_rows("muon_step_", params, grads, momenta, fast_bf16)
    _launch_muon(rows, (params, momenta), lr, momentum, nesterov, weight_decay, how)


def _launch_muon(rows, changed, lr, momentum, nesterov, weight_decay, how):
    if not rows:
        return
    table = array.array("q", itertools.chain.from_iterable(rows)).tobytes()
    like = changed[0][0]
    nbytes = nat.load().mqc_muon_workspace_bytes(table, len(rows))
    ws = _workspace(nbytes, "mqc_muon_step", like)
    lr = float(lr)
    nat.call("mqc_muon_step", like, table, len(rows), 1 - lr * weight_decay, lr, momentum, int(nesterov),
             *how, ws.data_ptr(), nbytes, nat.stream_of(like))
    nat.host().changed(changed)


class Muon(torch.optim.Optimizer):
    """Muon over the kernels of this module, for parameters that are matrices (embeddings, heads, norms and
    biases belong to an AdamW beside it). Momenta are fp32. fast_bf16: as orthogonalize's."""

    def __init__(self, params, lr: float = 1e-3, momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.1, steps: int = 5, coefficients=COEFFICIENTS,
                 eps: float = 1e-7, fast_bf16: bool = False):
        if lr < 0 or weight_decay < 0:
            raise ValueError(f"Muon: lr {lr} and weight_decay {weight_decay} are not negative")
        if not 0 <= momentum < 1:
            raise ValueError(f"Muon: momentum is in [0, 1), got {momentum}")
        _iteration("Muon", steps, coefficients, eps)
        super().__init__(params, {"lr": lr, "momentum": momentum, "nesterov": nesterov,
                                  "weight_decay": weight_decay, "steps": steps,
                                  "coefficients": tuple(coefficients), "eps": eps,
                                  "fast_bf16": fast_bf16})

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:  # (saved before there was one)
            group.setdefault("fast_bf16", False)

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() != 2:
                self.param_groups.pop()
                raise ValueError(f"Muon: parameters are matrices, got {tuple(p.shape)}")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work = []
        for group in self.param_groups:
            entries = []
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.layout != torch.strided:
                    raise ValueError("Muon: sparse gradients are not supported")
                g = p.grad.detach().contiguous().resolve_neg()
                s = self.state[p]
                if "momentum_buffer" not in s:
                    s["momentum_buffer"] = torch.zeros(p.shape, device=p.device, dtype=torch.float32)
                entries.append((p.detach(), g.to(p.dtype), s["momentum_buffer"]))
            if entries:
                work.append((group, entries))
        if not work:
            return loss
        lists = [list(x) for x in zip(*itertools.chain.from_iterable(e for _, e in work))]
        _muon_rows("Muon", *lists)  # no two in the same memory, over all groups
        for group, entries in work:
            params, grads, momenta = map(list, zip(*entries))
            how = _iteration("Muon", group["steps"], group["coefficients"], group["eps"])
            rows = _muon_rows("Muon", params, grads, momenta, group["fast_bf16"])
            _launch_muon(rows, (params, momenta), group["lr"], group["momentum"], group["nesterov"],
                         group["weight_decay"], how)
        return loss

    def load_state_dict(self, state_dict):
        """torch's loading casts momenta to the parameter's dtype: they are put back as they were saved."""
        super().load_state_dict(state_dict)
        ids = itertools.chain.from_iterable(g["params"] for g in state_dict["param_groups"])
        params = itertools.chain.from_iterable(g["params"] for g in self.param_groups)
        for i, p in zip(ids, params):
            saved = state_dict["state"].get(i)
            if saved is not None:
                self.state[p] = {k: v.detach().to(p.device, copy=True).contiguous()
                                 if isinstance(v, torch.Tensor) else v for k, v in saved.items()}
