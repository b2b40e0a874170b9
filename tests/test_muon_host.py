"""Refusals of orthogonalize and the Muon step, without a GPU."""
import array
import ctypes

import pytest
import torch

from mambaqc_amd import _native as nat
from mambaqc_amd.optim import Muon, muon_step_, orthogonalize

FAKE = ctypes.c_void_p(4096)  # never dereferenced: validation fails first


def test_orthogonalize_refuses():
    x = torch.zeros(3, 4)
    with pytest.raises(ValueError, match="rows, cols"):
        orthogonalize(torch.zeros(4))
    with pytest.raises(ValueError, match="steps"):
        orthogonalize(x, steps=0)
    with pytest.raises(ValueError, match="three coefficients"):
        orthogonalize(x, coefficients=(1.5, -0.5))
    with pytest.raises(ValueError, match="eps"):
        orthogonalize(x, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        orthogonalize(x, eps=float("nan"))
    with pytest.raises(TypeError, match="dtype"):
        orthogonalize(x.double())
    with pytest.raises(RuntimeError, match="ROCm device"):
        orthogonalize(x)


def test_muon_refuses():
    p, v = torch.zeros(3, 4), torch.zeros(4)
    with pytest.raises(ValueError, match="lengths"):
        muon_step_([p], [p, p], [p])
    with pytest.raises(ValueError, match="matrices"):
        muon_step_([v], [v], [v])
    with pytest.raises(ValueError, match="gradient is"):
        muon_step_([p], [p.half()], [p])
    with pytest.raises(ValueError, match="momenta"):
        muon_step_([p.requires_grad_()], [p], [p.half()])
    with pytest.raises(RuntimeError, match="ROCm device"):
        muon_step_([p], [p], [p])
    with pytest.raises(ValueError, match="steps"):
        muon_step_([p], [p], [p], steps=101)
    param = torch.nn.Parameter
    with pytest.raises(ValueError, match="matrices"):
        Muon([param(v)])
    opt = Muon([param(torch.zeros(2, 3))])
    with pytest.raises(ValueError, match="matrices"):
        opt.add_param_group({"params": [param(v)]})
    assert len(opt.param_groups) == 1
    for bad in ({"lr": -1}, {"weight_decay": -1}, {"momentum": 1.0}, {"steps": 0}, {"eps": -1}, {"coefficients": ()}):
        with pytest.raises(ValueError):
            Muon([param(torch.zeros(2, 3))], **bad)
    q = param(torch.zeros(2, 3))
    opt = Muon([q])
    opt.step()
    q.grad = torch.zeros(2, 3)
    with pytest.raises(RuntimeError, match="ROCm device"):
        opt.step()


def test_validation_codes():
    lib = nat.load()
    f = lambda b=1, r=3, c=4, steps=5, eps=0.0, dtype=0, ptr=FAKE, ws=1 << 40, at=FAKE: lib.mqc_orthogonalize(
        ptr, FAKE, b, r, c, steps, 1.0, 1.0, 1.0, eps, dtype, at, ws, None)
    assert f(b=-1) == -2 and f(r=0) == -2 and f(c=0) == -2 and f(steps=0) == -2 and f(steps=101) == -2
    assert f(eps=-1.0) == -2 and f(eps=float("nan")) == -2
    assert f(dtype=3) == -3 and f(ptr=None) == -1 and f(at=None) == -1 and f(ws=10) == -6
    assert f(at=ctypes.c_void_p(4096 + 128)) == -4
    assert f(b=65536) == -5 and f(r=32769, c=32769) == -5 and f(r=(1 << 24) + 1) == -5
    assert f(b=0, ptr=None) == 0
    size = lib.mqc_orthogonalize_workspace_bytes
    assert size(1, 0, 3, 0) == -2 and size(1, 3, 3, 4) == -3 and size(2, 64, 64, 1) > size(1, 64, 64, 1) > 0
    assert size(1, 512, 300, 0) > size(1, 512, 300, 1) and size(1, 64, 64, 0) == size(1, 64, 64, 1)
    row = [4096, 4096, 4096, 3, 4, 0]

    def step(rows, ws=1 << 40, at=FAKE, steps=5):
        table = array.array("q", [v for r in rows for v in r]).tobytes()
        return lib.mqc_muon_step(table, len(rows), 1.0, 1.0, 0.9, 1, steps, 1.0, 1.0, 1.0, 0.0, at, ws, None)

    for i, bad, code in ((0, 0, -1), (1, 0, -1), (2, 0, -1), (3, 0, -2), (4, -1, -2), (5, 9, -3), (3, 1 << 25, -5)):
        assert step([row, row[:i] + [bad] + row[i + 1:]]) == code
    assert step([row], steps=0) == -2 and step([row], at=None) == -1 and step([row], ws=64) == -6
    assert step([]) == 0
    assert lib.mqc_muon_step(None, 1, 1.0, 1.0, 0.9, 1, 5, 1.0, 1.0, 1.0, 0.0, FAKE, 1 << 40, None) == -1
    assert lib.mqc_muon_step(None, -1, 1.0, 1.0, 0.9, 1, 5, 1.0, 1.0, 1.0, 0.0, FAKE, 1 << 40, None) == -2
    table = array.array("q", row * 3).tobytes()
    assert lib.mqc_muon_workspace_bytes(table, 3) > lib.mqc_muon_workspace_bytes(table, 1) > 0
    # Launches of 2^32 threads are refused before the first: nothing of the table is done.
    big = [4096, 4096, 4096, 32768, 1 << 24, 1]
    assert f(r=32768, c=1 << 24, dtype=1, ws=1 << 62) == -5
    assert step([row, big], ws=1 << 62) == -5 and step([big, row], ws=1 << 62) == -5


def test_pairs_for_every_type():
    """The C interface's choice for bf16 matrices: as much room as fp32's take; none for the other types."""
    size = nat.load().mqc_orthogonalize_workspace_bytes
    assert size(1, 512, 300, 17) == size(1, 512, 300, 0) == size(1, 512, 300, 16) == size(1, 512, 300, 18)
    assert size(1, 512, 300, 1) < size(1, 512, 300, 17) and size(1, 64, 64, 1) == size(1, 64, 64, 17)
    for bad in (-1, 3, 15, 19, 32, 33):
        assert size(1, 512, 300, bad) == -3
    room = nat.load().mqc_muon_workspace_bytes
    table = lambda dtype: array.array("q", [4096, 4096, 4096, 512, 300, dtype]).tobytes()
    assert room(table(1), 1) < room(table(17), 1) == room(table(0), 1) and room(table(19), 1) == -3
    both = array.array("q", [4096, 4096, 4096, 512, 300, 1, 4096, 4096, 4096, 512, 300, 17]).tobytes()
    assert room(both, 2) == room(table(17), 1)


def test_groups_saved_without_the_choice():
    p = torch.nn.Parameter(torch.zeros(2, 3))
    opt = Muon([p], fast_bf16=True)
    saved = opt.state_dict()
    assert saved["param_groups"][0].pop("fast_bf16") is True
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["fast_bf16"] is False
