"""layer_norm's refusals and shape rules, without a GPU."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mambaqc_amd  # noqa: F401  (registers torch.ops.mambaqc.*)
from mambaqc_amd import _native as nat
from mambaqc_amd.kernels import layer_norm
from mambaqc_amd.layers import LayerNorm

FAKE = ctypes.c_void_p(4096)  # never dereferenced: validation fails first


def test_refuses_shapes_types_and_devices():
    x, w = torch.zeros(2, 3, 4), torch.zeros(4)
    for call in (layer_norm, torch.ops.mambaqc.layer_norm):
        with pytest.raises(ValueError, match="no axis"):
            call(torch.zeros(()))
        with pytest.raises(ValueError, match="weight"):
            call(x, torch.zeros(3))
        with pytest.raises(ValueError, match="bias"):
            call(x, w, torch.zeros(1, 4))
        with pytest.raises(RuntimeError, match="ROCm device"):
            call(x, w)
    with pytest.raises(ValueError, match="last axis"):
        LayerNorm((3, 4))
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            layer_norm(torch.autograd.forward_ad.make_dual(x, x), w)


def test_module_is_a_layer_norm():
    m = LayerNorm(6, eps=1e-3)
    assert isinstance(m, torch.nn.LayerNorm) and sorted(m.state_dict()) == ["bias", "weight"]
    assert sorted(LayerNorm(6, bias=False).state_dict()) == ["weight"]
    assert not LayerNorm(6, elementwise_affine=False).state_dict()


def test_validation_codes():
    lib = nat.load()
    widest = lib.mqc_layer_norm_max_width()
    assert widest == 8192
    fwd = lambda rows, d, row=None, dtype=0, ptr=FAKE: lib.mqc_layer_norm_fwd(
        ptr, d if row is None else row, None, None, FAKE, None, rows, d, 1e-5, dtype, None)
    assert fwd(-1, 4) == -2 and fwd(2, 0) == -2 and fwd(2, 4, row=3) == -2
    assert fwd(2, 4, dtype=3) == -3 and fwd(2, 4, ptr=None) == -1
    assert fwd(2, widest + 1) == -5 and fwd(1 << 31, 4) == -5 and fwd(1 << 27, 1024) == -5
    assert fwd(0, 4, ptr=None) == 0
    bwd = lambda rows, d, ws=1 << 40, ptr=FAKE, at=FAKE, dw=FAKE: lib.mqc_layer_norm_bwd(
        FAKE, d, None, ptr, FAKE, FAKE, dw, dw, rows, d, 1, at, ws, None)
    assert bwd(0, 4) == -2 and bwd(2, 4, ptr=None) == -1 and bwd(2, 4, at=None) == -1
    assert bwd(2, 4, ws=5) == -6 and bwd(2, widest + 1) == -5
    assert lib.mqc_layer_norm_workspace_bytes(0, 4) == -2
    assert lib.mqc_layer_norm_workspace_bytes(1, widest + 1) == -5
    assert lib.mqc_layer_norm_workspace_bytes(1, 5) == 40


def test_fake_kernels():
    with FakeTensorMode():
        x = torch.empty(2, 7, 6, device="cuda", dtype=torch.bfloat16)
        y, stats = torch.ops.mambaqc.layer_norm(x, torch.empty(6, device="cuda"))
        assert y.shape == x.shape and y.dtype == x.dtype and stats.shape == (14, 2)


def test_too_wide_a_module_is_refused_as_it_is_made():
    from mambaqc_amd.kernels.norm import MAX_WIDTH

    assert MAX_WIDTH == nat.load().mqc_layer_norm_max_width()
    assert LayerNorm(MAX_WIDTH).normalized_shape == (MAX_WIDTH,)
    with pytest.raises(ValueError, match="at most 8192"):
        LayerNorm(MAX_WIDTH + 1)
