"""gate_norm_residual's refusals and shape rules, without a GPU."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mambaqc_amd  # noqa: F401  (registers torch.ops.mambaqc.*)
from mambaqc_amd import _native as nat
from mambaqc_amd.kernels import gate_norm_residual
from mambaqc_amd.kernels.gate_norm import _z_rows

FAKE = ctypes.c_void_p(4096)  # never dereferenced: validation fails first


def test_refuses_shapes_types_and_devices():
    x, w = torch.zeros(2, 3, 4), torch.zeros(4)
    how = {"scale": w, "pre_weight": w}
    with pytest.raises(ValueError, match="one shape"):
        gate_norm_residual(x, x[:1], **how)
    with pytest.raises(ValueError, match="one shape"):
        gate_norm_residual(torch.zeros(()), torch.zeros(()), **how)
    with pytest.raises(ValueError, match="z must be"):
        gate_norm_residual(x, x, torch.zeros(2, 3, 8), **how)
    for name in ("scale", "pre_weight", "post_weight"):
        with pytest.raises(ValueError, match=name):
            gate_norm_residual(x, x, **{**how, name: torch.zeros(3)})
    with pytest.raises(RuntimeError, match="ROCm device"):
        gate_norm_residual(x, x, x, **how)
    with pytest.raises(RuntimeError, match="ROCm device"):
        gate_norm_residual(x.requires_grad_(), x, x, **how)


def test_validation_codes():
    lib = nat.load()
    widest = lib.mqc_gate_norm_max_width()
    assert widest == 8192
    fwd = lambda rows, d, row=None, dtype=0, ptr=FAKE: lib.mqc_gate_norm_fwd(
        ptr, FAKE, FAKE, d if row is None else row, FAKE, FAKE, FAKE, FAKE, FAKE, None, rows, d, 1e-6,
        dtype, None)
    assert fwd(-1, 4) == -2 and fwd(2, 0) == -2 and fwd(2, 4, row=3) == -2
    assert fwd(2, 4, dtype=3) == -3 and fwd(2, 4, ptr=None) == -1
    assert fwd(2, widest + 1) == -5 and fwd(1 << 31, 4) == -5
    assert fwd(0, 4, ptr=None) == 0
    bwd = lambda rows, d, ws=1 << 40, ptr=FAKE, dz=FAKE: lib.mqc_gate_norm_bwd(
        FAKE, FAKE, FAKE, d, FAKE, FAKE, FAKE, ptr, None, None, FAKE, FAKE, dz, FAKE, FAKE, FAKE, rows,
        d, 1, FAKE, ws, None)
    assert bwd(0, 4) == -2 and bwd(2, 4, ptr=None) == -1 and bwd(2, 4, dz=None) == -1
    assert bwd(2, 4, ws=5) == -6 and bwd(2, widest + 1) == -5
    assert lib.mqc_gate_norm_workspace_bytes(0, 4) == -2
    assert lib.mqc_gate_norm_workspace_bytes(1, widest + 1) == -5
    assert lib.mqc_gate_norm_workspace_bytes(1, 5) == 60


def test_z_read_in_place():
    wide = torch.zeros(3, 5, 24)
    for part in (wide[..., :8], wide[..., 8:16], wide[1, :, 16:], wide[:1, 2:4, 3:9], wide[0, 0, :7]):
        view, row = _z_rows(part, torch.float32)
        assert view.data_ptr() == part.data_ptr() and row >= part.shape[-1]
    assert _z_rows(wide[:, 1:2, :8], torch.float32)[1] == 5 * 24
    for part in (wide[:, 1:3, :8], wide.transpose(0, 1), wide[..., ::2], wide[:1].expand(3, -1, -1),
                 wide[:, :1].expand(-1, 5, -1)):
        view, row = _z_rows(part, torch.float32)
        assert view.is_contiguous() and row == part.shape[-1]


def test_fake_kernels():
    with FakeTensorMode():
        x = torch.empty(2, 7, 6, device="cuda", dtype=torch.bfloat16)
        w = torch.empty(6, device="cuda")
        out, n, stats = torch.ops.mambaqc.gate_norm_residual(x, x.float(), x, None, w, w)
        assert out.shape == n.shape == x.shape and out.dtype == n.dtype == torch.float32
        assert stats.shape == (14, 2)
        grads = torch.ops.mambaqc.gate_norm_residual_backward(x, x, None, w, w, w, stats, x, x)
        assert grads[0].dtype == torch.bfloat16 and grads[2].numel() == 0
        assert all(g.shape == (6,) and g.dtype == torch.float32 for g in grads[3:])


def test_registered_operators_check_their_arguments():
    """torch.ops.mambaqc.gate_norm_residual* refuse what gate_norm_residual refuses."""
    x, w = torch.zeros(2, 3, 4), torch.zeros(4)
    for op, rest in ((torch.ops.mambaqc.gate_norm_residual, ()),
                     (torch.ops.mambaqc.gate_norm_residual_backward, (torch.zeros(6, 2), x, x))):
        with pytest.raises(ValueError, match="one shape"):
            op(x, x[:1], None, None, w, w, *rest)
        with pytest.raises(ValueError, match="z must be"):
            op(x, x, x[..., :2], None, w, w, *rest)
        for bad in ((w[:3], w, w), (w, w[:3], w), (w, w, w[:3])):
            with pytest.raises(ValueError, match="must be \\[4\\]"):
                op(x, x, x, *bad, *rest)


@pytest.mark.parametrize("which", range(6))
def test_refuses_forward_mode(which):
    """A tangent would be lost: the kernels see the values alone."""
    ops = [torch.zeros(3, 4) for _ in range(3)] + [torch.zeros(4) for _ in range(3)]
    with torch.autograd.forward_ad.dual_level():
        ops[which] = torch.autograd.forward_ad.make_dual(ops[which], torch.ones_like(ops[which]))
        x, y, gate, post, scale, pre = ops
        with pytest.raises(NotImplementedError, match="forward-mode"):
            gate_norm_residual(x, y, gate, scale=scale, pre_weight=pre, post_weight=post)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.ops.mambaqc.gate_norm_residual(*ops)


def test_negated_views_are_read_as_what_they_stand_for():
    gate = torch.randn(5, 1, dtype=torch.complex64).conj().imag
    view, row = _z_rows(gate, torch.float32)
    assert gate.is_neg() and not view.is_neg() and torch.equal(view, gate) and row == view.stride(0)


@pytest.mark.parametrize("d,rows", [(1, 16 << 24), (64, 16 << 24), (65, 8 << 24), (128, 8 << 24), (129, 4 << 24),
                                    (1024, 4 << 24), (1025, 1 << 25), (8192, 1 << 23)])
def test_rows_past_one_launch_are_refused(d, rows):
    """2^32 threads and more along an axis, which HIP does not launch. (Without pointers: what is within
    the limit is refused for those.)"""
    fwd = lambda rows: nat.load().mqc_gate_norm_fwd(None, None, None, 0, None, None, None, None, None, None,
                                                    rows, d, 1e-6, 0, None)
    assert fwd(rows) == -5 and fwd(rows - 16) == -1
