"""The gated delta rule's refusals and shape rules, without a GPU."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mambaqc_amd  # noqa: F401  (registers torch.ops.mambaqc.*)
from mambaqc_amd import _native as nat
from mambaqc_amd.kernels import gated_delta, gated_delta_step_

FAKE = ctypes.c_void_p(4096)  # never dereferenced: validation fails first
NINE = (ctypes.c_int64 * 9)()


def z(*shape, **kw):
    return torch.zeros(*shape, **kw)


def operands(b=2, t=3, hk=1, hv=2, dk=4, dv=5):
    return [z(b, t, hk, dk), z(b, t, hk, dk), z(b, t, hv, dv), z(b, t, hv), z(b, t, hv)]


BAD = [({"q": z(2, 3, 1, 5)}, "q and k are"), ({"k": z(2, 3, 4)}, "q and k are"), ({"v": z(2, 4, 2, 5)}, "q and k are"),
       ({"q": z(2, 3, 4), "k": z(2, 3, 4)}, "q and k are"), ({"v": z(2, 3, 10)}, "q and k are"),
       ({"q": z(2, 3, 3, 4), "k": z(2, 3, 3, 4)}, "not a multiple"),
       ({"q": z(2, 3, 0, 4), "k": z(2, 3, 0, 4)}, "not a multiple"),
       ({"q": z(2, 3, 1, 0), "k": z(2, 3, 1, 0)}, "not a multiple"),
       ({"v": z(2, 3, 2, 0)}, "not a multiple"),
       ({"q": z(2, 3, 1, 129), "k": z(2, 3, 1, 129)}, "at most 128"),
       ({"log_decay": z(2, 3)}, "log_decay"), ({"beta": z(2, 3, 1)}, "beta"),
       ({"h0": z(2, 2, 5, 4)}, "state"), ({"h0": z(1, 2, 4, 5)}, "state"),
       ({"reset": z(2, 3)}, "reset"), ({"reset": z(3, 2, dtype=torch.bool)}, "reset")]


@pytest.mark.parametrize("change,match", BAD)
def test_refuses_shapes(change, match):
    args = dict(zip(("q", "k", "v", "log_decay", "beta"), operands())) | {"h0": None, "reset": None}
    args |= change
    with pytest.raises(ValueError, match=match):
        gated_delta(**args)
    for op in (torch.ops.mambaqc.gated_delta, torch.ops.mambaqc.gated_delta_train):
        with pytest.raises(ValueError, match=match):
            op(*args.values())


def test_refuses_devices_types_and_steps():
    ops = operands()
    with pytest.raises(RuntimeError, match="ROCm device"):
        gated_delta(*ops)
    with pytest.raises(RuntimeError, match="ROCm device"):
        gated_delta(ops[0].requires_grad_(), *ops[1:])
    h = z(2, 2, 4, 5)
    with pytest.raises(ValueError, match="one token"):
        gated_delta_step_(*operands(), h)
    one = operands(t=1)
    for bad in (h.half(), z(2, 2, 5, 4).transpose(2, 3), torch._neg_view(h)):
        with pytest.raises(ValueError, match="contiguous float32"):
            gated_delta_step_(*one, bad)
    with pytest.raises(RuntimeError, match="ROCm device"):
        gated_delta_step_(*one, h)


@pytest.mark.parametrize("which", range(6))
def test_refuses_forward_mode(which):
    ops = operands(t=1) + [z(2, 2, 4, 5)]
    with torch.autograd.forward_ad.dual_level():
        ops[which] = torch.autograd.forward_ad.make_dual(ops[which], torch.ones_like(ops[which]))
        for call in (lambda: gated_delta(*ops[:5], h0=ops[5]), lambda: gated_delta_step_(*ops),
                     lambda: torch.ops.mambaqc.gated_delta(*ops, None)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


def test_validation_codes():
    lib = nat.load()

    def fwd(b=2, t=3, hk=1, hv=2, dk=4, dv=5, dtype=0, gt=0, bt=0, ptr=FAKE, ws=1 << 40, at=FAKE, saved=None):
        return lib.mqc_gated_delta_fwd(ptr, FAKE, FAKE, NINE, FAKE, gt, FAKE, bt, None, None, FAKE, FAKE,
                                       saved, saved, b, t, hk, hv, dk, dv, 1.0, dtype, at, ws, None)

    def bwd(b=2, t=3, hk=1, hv=2, dk=4, dv=5, ptr=FAKE, ws=1 << 40):
        return lib.mqc_gated_delta_bwd(FAKE, FAKE, FAKE, NINE, FAKE, 0, FAKE, 0, None, ptr, FAKE, FAKE, None,
                                       FAKE, FAKE, FAKE, FAKE, FAKE, None, b, t, hk, hv, dk, dv, 1.0, 0,
                                       FAKE, ws, None)

    def step(b=2, hk=1, hv=2, dk=4, dv=5, ptr=FAKE, dtype=0):
        return lib.mqc_gated_delta_step(FAKE, FAKE, FAKE, NINE, FAKE, 0, FAKE, 0, ptr, FAKE, b, hk, hv, dk,
                                        dv, 1.0, dtype, None)

    for f in (fwd, bwd, step):
        assert f(b=-1) == -2 and f(hk=0) == -2 and f(hv=0) == -2 and f(hk=2, hv=3) == -2
        assert f(dk=0) == -2 and f(dv=0) == -2
        assert f(dk=129) == -5 and f(dv=(1 << 20) + 1) == -5 and f(b=1 << 24, hv=64) == -5
        assert f(ptr=None) == -1
    assert fwd(t=-1) == -2 and fwd(dtype=3) == -3 and fwd(gt=4) == -3 and fwd(bt=-1) == -3
    assert fwd(ws=100) == -6 and fwd(at=ctypes.c_void_p(4100)) == -4 and fwd(saved=ctypes.c_void_p(4100)) == -4
    assert fwd(b=0, ptr=None) == 0 and step(b=0, ptr=None) == 0 and step(dtype=7) == -3
    assert bwd(b=0) == -2 and bwd(t=0) == -2 and bwd(ws=100) == -6
    assert fwd(t=(1 << 31) + 1) == -5 and fwd(b=1 << 10, t=1 << 31) == -5
    # 2^32 threads: chunks of a head, columns of 16.
    assert fwd(b=1, hk=1, hv=1, t=64 << 24, ptr=None) == -5 and fwd(b=1, hk=1, hv=1, t=63 << 24, ptr=None) == -1
    # (in the backward, and in a forward that stores what it reads, four times as many for chunks)
    assert bwd(b=1, hk=1, hv=1, t=64 << 22, ptr=None) == -5 and bwd(b=1, hk=1, hv=1, t=63 << 22, ptr=None) == -1
    assert fwd(b=1, hk=1, hv=1, t=64 << 22, ptr=None, saved=FAKE) == -5
    assert fwd(b=1, hk=1, hv=1, t=63 << 22, ptr=None, saved=FAKE) == -1
    assert step(b=1 << 20, hv=1, dv=256, ptr=None) == -5 and step(b=1 << 19, hv=1, dv=256, ptr=None) == -1
    size = lib.mqc_gated_delta_workspace_bytes
    assert size(-1, 1, 1, 1, 1, 1, 0, 0) == -2 and size(1, 1, 1, 1, 200, 1, 0, 0) == -5
    assert 0 < size(1, 64, 1, 1, 32, 32, 1, 0) < size(1, 64, 1, 1, 32, 32, 0, 0) < size(1, 64, 1, 1, 32, 32, 0, 1)
    assert [lib.mqc_gated_delta_key_width(n) for n in (0, 1, 32, 33, 64, 65, 128, 129)] == [
        -2, 32, 32, 64, 64, 128, 128, -5]
    assert [lib.mqc_gated_delta_value_width(n) for n in (0, 1, 32, 33, 500)] == [-2, 32, 32, 64, 512]


def test_fake_kernels():
    with FakeTensorMode():
        e = lambda *s, dtype=torch.float32: torch.empty(*s, device="cuda", dtype=dtype)
        q, v = e(2, 70, 1, 40, dtype=torch.bfloat16), e(2, 70, 3, 50)
        gates = e(2, 70, 3)
        o, h = torch.ops.mambaqc.gated_delta(q, q, v, gates, gates)
        assert o.shape == v.shape and o.dtype == torch.float32 and h.shape == (2, 3, 40, 50)
        o, h, states, resid = torch.ops.mambaqc.gated_delta_train(q, q, v.bfloat16(), gates, gates)
        assert o.dtype == torch.bfloat16 and states.shape == (2, 3, 2, 64, 64)
        assert resid.shape == (2, 3, 2, 64, 64) and resid.dtype == torch.float32
