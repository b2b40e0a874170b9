"""The gated scan's refusals and shape rules, without a GPU."""
import ctypes
import shutil
import subprocess
import sys

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mambaqc_amd  # noqa: F401  (registers torch.ops.mambaqc.*)
from mambaqc_amd import _native as nat
from mambaqc_amd.kernels import gated_scan, gated_scan_step_
from mambaqc_amd.kernels.gated import _rows

FAKE = ctypes.c_void_p(4096)  # never dereferenced: validation fails first


def z(*shape, **kw):
    return torch.zeros(*shape, **kw)


def test_refuses_shapes_types_and_devices():
    x, lam = z(2, 3, 4), z(4)
    with pytest.raises(ValueError, match="one shape"):
        gated_scan(z(2, 3, 5), x, x, lam)
    with pytest.raises(ValueError, match="one shape"):
        gated_scan(z(3, 4), z(3, 4), z(3, 4), lam)
    with pytest.raises(ValueError, match="log_rate"):
        gated_scan(x, x, x, z(3))
    with pytest.raises(ValueError, match="state"):
        gated_scan(x, x, x, lam, h0=z(2, 3, 4))
    with pytest.raises(ValueError, match="reset"):
        gated_scan(x, x, x, lam, reset=z(2, 3))
    with pytest.raises(ValueError, match="reset"):
        gated_scan(x, x, x, lam, reset=z(2, 4, dtype=torch.bool))
    with pytest.raises(RuntimeError, match="ROCm device"):
        gated_scan(x, x, x, lam)
    with pytest.raises(RuntimeError, match="ROCm device"):
        gated_scan(x.requires_grad_(), x, x, lam)
    with pytest.raises(ValueError, match="one token"):
        gated_scan_step_(x, x, x, lam, z(2, 4))
    one = z(2, 1, 4)
    with pytest.raises(ValueError, match="contiguous float32"):
        gated_scan_step_(one, one, one, lam, z(2, 4, dtype=torch.float16))
    with pytest.raises(ValueError, match="contiguous float32"):
        gated_scan_step_(one, one, one, lam, z(4, 2).T)
    with pytest.raises(RuntimeError, match="ROCm device"):
        gated_scan_step_(one, one, one, lam, z(2, 4))


def test_validation_codes():
    lib = nat.load()
    fwd = lambda b, t, d, row=None, dtype=0, ptr=FAKE, ws=1 << 40: lib.mqc_gated_scan_fwd(
        ptr, d if row is None else row, FAKE, d, FAKE, d, FAKE, None, None, FAKE, FAKE, None, b, t, d,
        dtype, FAKE, ws, None)
    assert fwd(-1, 3, 4) == -2 and fwd(1, -3, 4) == -2 and fwd(1, 3, -4) == -2
    assert fwd(2, 3, 4, row=3) == -2
    assert fwd(2, 3, 4, dtype=5) == -3
    assert fwd(2, 3, 4, ptr=None) == -1
    assert fwd(1 << 20, 3, 4) == -5
    assert fwd(2, 3, 4, ws=3) == -6
    assert fwd(0, 3, 4, ptr=None) == 0 and fwd(2, 3, 0, ptr=None) == 0
    bwd = lambda b, t, d, ws=1 << 40, ptr=FAKE: lib.mqc_gated_scan_bwd(
        FAKE, d, FAKE, d, FAKE, d, FAKE, None, ptr, FAKE, None, FAKE, FAKE, FAKE, FAKE, None, b, t, d,
        0, FAKE, ws, None)
    assert bwd(0, 3, 4) == -2 and bwd(2, 0, 4) == -2 and bwd(2, 3, 0) == -2
    assert bwd(2, 3, 4, ws=3) == -6 and bwd(2, 3, 4, ptr=None) == -1
    step = lambda b, d, ptr=FAKE, dtype=0: lib.mqc_gated_scan_step(
        FAKE, d, FAKE, d, FAKE, d, FAKE, ptr, FAKE, b, d, dtype, None)
    assert step(2, 4, ptr=None) == -1 and step(2, 4, dtype=3) == -3 and step(-2, 4) == -2
    assert step(0, 4) == 0
    assert lib.mqc_gated_scan_workspace_bytes(-1, 1, 1) == -2


def test_rows_read_in_place():
    wide = z(3, 5, 24)
    for part in (wide[..., :8], wide[..., 8:], wide[:, :1, 4:9], wide[:1, 2:4, 4:9]):
        view, row = _rows(part, torch.float32)
        assert view.data_ptr() == part.data_ptr()
        assert row >= part.shape[2]
    assert _rows(wide[:, 1:2, :8], torch.float32)[1] == 5 * 24  # one token a sequence
    for part in (wide[:, 1:3, :8], wide.transpose(0, 1), wide[..., ::2], wide[:1].expand(3, -1, -1)):
        view, row = _rows(part, torch.float32)
        assert view.is_contiguous() and row == part.shape[2]


def test_fake_kernels():
    with FakeTensorMode():
        x = torch.empty(2, 70, 6, device="cuda", dtype=torch.bfloat16)
        lam, h0 = torch.empty(6, device="cuda"), torch.empty(2, 6, device="cuda")
        y, h = torch.ops.mambaqc.gated_scan(x, x, x.float(), lam, h0, None)
        assert y.shape == (2, 70, 6) and y.dtype == torch.float32 and h.shape == (2, 6)
        y, h, carries = torch.ops.mambaqc.gated_scan_train(x, x, x, lam, None, None)
        assert y.dtype == torch.bfloat16 and carries.dtype == torch.float32
        every = nat.load().mqc_gated_scan_chunk()
        assert carries.shape == (2, -(-70 // every), 6)


def test_registered_operators_check_their_arguments():
    """torch.ops.mambaqc.gated_scan* refuse what gated_scan refuses, before anything reads it."""
    x, lam, h = z(2, 3, 4), z(4), z(2, 4)
    ops = torch.ops.mambaqc
    for op in (ops.gated_scan, ops.gated_scan_train):
        with pytest.raises(ValueError, match="one shape"):
            op(z(1, 3, 4), x, x, lam, None, None)
        with pytest.raises(ValueError, match="one shape"):
            op(z(3, 4), z(3, 4), z(3, 4), lam, None, None)
        with pytest.raises(ValueError, match="log_rate"):
            op(x, x, x, z(3), None, None)
        with pytest.raises(ValueError, match="state"):
            op(x, x, x, lam, z(1, 4), None)
        with pytest.raises(ValueError, match="reset"):
            op(x, x, x, lam, None, z(2, 3, dtype=torch.int32))
    with pytest.raises(ValueError, match="one shape"):
        ops.gated_scan_backward(x, x, z(2, 9, 4), lam, None, z(2, 1, 4), x, h)
    with pytest.raises(ValueError, match="reset"):
        ops.gated_scan_backward(x, x, x, lam, z(2, 2, dtype=torch.bool), z(2, 1, 4), x, h)


@pytest.mark.parametrize("which", range(5))
def test_refuses_forward_mode(which):
    """A tangent would be lost: the kernels see the values alone."""
    ops = [z(2, 1, 4) for _ in range(3)] + [z(4), z(2, 4)]
    with torch.autograd.forward_ad.dual_level():
        ops[which] = torch.autograd.forward_ad.make_dual(ops[which], torch.ones_like(ops[which]))
        calls = [lambda: gated_scan(*ops[:4], h0=ops[4]), lambda: gated_scan_step_(*ops),
                 lambda: torch.ops.mambaqc.gated_scan(*ops, None),
                 lambda: torch.ops.mambaqc.gated_scan_train(*ops, None)]
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_negated_views_are_read_as_what_they_stand_for():
    x = torch.randn(2, 3, 1, dtype=torch.complex64).conj().imag
    view, row = _rows(x, torch.float32)
    assert x.is_neg() and not view.is_neg() and torch.equal(view, x) and row == view.stride(1)
    one = z(2, 1, 4)
    with pytest.raises(ValueError, match="contiguous float32"):
        gated_scan_step_(one, one, one, z(4), torch._neg_view(z(2, 4)))


def test_sizes_past_one_launch_are_refused():
    """2^32 threads and more along an axis, which HIP does not launch. (Without pointers: what is within
    the limit is refused for those.)"""
    lib = nat.load()
    fwd = lambda b, t, d: lib.mqc_gated_scan_fwd(None, d, None, d, None, d, None, None, None, None, None,
                                                 None, b, t, d, 0, None, 0, None)
    bwd = lambda b, t, d: lib.mqc_gated_scan_bwd(None, d, None, d, None, d, None, None, None, None, None,
                                                 None, None, None, None, None, b, t, d, 0, None, 0, None)
    for walk in (fwd, bwd):
        assert walk(65535, 32768, 1) == -5 and walk(65535, 16384, 1) == -1
        assert walk(65535, 1, 1 << 31) == -5 and walk(1, 1 << 31, 64) == -5
        assert walk(1, 1 << 29, 64) == -1
    assert fwd(65535, 1, 16384) == -1 and fwd(65535, 16, 65536) == -1  # (of short sequences few waves)
    step = lambda b, d: lib.mqc_gated_scan_step(None, d, None, d, None, d, None, None, None, b, d, 0, None)
    assert step(65535, 1 << 31) == -1 and step(65536, 1) == -5


def test_host_module_tells_what_it_was_compiled_against(tmp_path):
    """Beside a library of another version, _host.abi() still gives its own, so that a stale module shows."""
    other = tmp_path / "other.c"
    other.write_text("int mqc_abi_version(void) { return 99; }")
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    subprocess.run([cc, "-shared", "-fPIC", str(other), "-o", str(tmp_path / "other.so")], check=True)
    code = ("import ctypes, importlib.util, sys, torch; ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)\n"
            "spec = importlib.util.spec_from_file_location('_host', sys.argv[2])\n"
            "module = importlib.util.module_from_spec(spec); spec.loader.exec_module(module)\n"
            "print(module.abi())")
    out = subprocess.run([sys.executable, "-c", code, str(tmp_path / "other.so"),
                          str(nat.LIB_PATH.parent / "_host.so")], capture_output=True, text=True, check=True)
    assert int(out.stdout) == nat.ABI_VERSION
