"""The AdamW step's refusals and argument checks, without a GPU."""
import copy
import ctypes
import pickle
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from mambaqc_amd import _native as nat
from mambaqc_amd.optim import AdamW, adamw8_step_, adamw_step_, grad_norm, state_blocks

E4M3 = torch.float8_e4m3fn


def rows(*values):
    return (ctypes.c_int64 * max(1, len(values)))(*values)


def test_refuses_lists_that_do_not_match():
    t = [torch.ones(6)]
    with pytest.raises(ValueError, match="lengths"):
        adamw_step_(t, [], [], [], step=1)
    with pytest.raises(ValueError, match="states"):
        adamw_step_(t, t, [torch.ones(5)], t, step=1)
    with pytest.raises(ValueError, match="states"):
        adamw_step_(t, t, t, [torch.ones(6, dtype=torch.float16)], step=1)
    with pytest.raises(ValueError, match="gradient"):
        adamw_step_(t, [torch.ones(6, dtype=torch.float16)], t, t, step=1)
    with pytest.raises(ValueError, match="gradient"):
        adamw_step_(t, [torch.ones(2, 3)], t, t, step=1)
    with pytest.raises(ValueError, match="contiguous"):
        adamw_step_([torch.ones(12)[::2]], t, t, t, step=1)
    with pytest.raises(TypeError, match="unsupported dtype"):
        d = [torch.ones(6, dtype=torch.float64)]
        adamw_step_(d, d, t, t, step=1)
    with pytest.raises(ValueError, match="count from 1"):
        adamw_step_(t, t, t, t, step=0)
    with pytest.raises(RuntimeError, match="ROCm device"):
        adamw_step_(t, t, t, t, step=1)
    assert adamw_step_([], [], [], [], step=1) is None


def test_refuses_8_bit_states_that_do_not_match():
    t, s = [torch.ones(300)], [torch.ones(2)]
    c = [torch.zeros(300, dtype=torch.uint8).view(E4M3)]
    assert state_blocks(300) == 2 and state_blocks(0) == 0 and state_blocks(256) == 1
    with pytest.raises(ValueError, match="states"):
        adamw8_step_(t, t, t, s, c, s, step=1)
    with pytest.raises(ValueError, match="scales"):
        adamw8_step_(t, t, c, [torch.ones(1)], c, s, step=1)
    with pytest.raises(ValueError, match="scales"):
        adamw8_step_(t, t, c, s, c, [torch.ones(3)], step=1)
    with pytest.raises(RuntimeError, match="ROCm device"):
        adamw8_step_(t, t, c, s, c, s, step=1)


def test_optimizer_arguments():
    p = torch.nn.Parameter(torch.ones(3))
    for bad in ({"lr": -1.0}, {"betas": (1.0, 0.9)}, {"state_bits": 16}, {"eps": -1e-8},
                {"weight_decay": -0.1}):
        with pytest.raises(ValueError):
            AdamW([p], **bad)
    opt = AdamW([p])
    assert opt.step() is None  # nothing has a gradient
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="ROCm device"):
        opt.step()
    with pytest.raises(ValueError, match="no tensors"):
        grad_norm([])


def test_validation_codes():
    lib, how = nat.load(), [1.0] * 8
    step = lambda *v, count=1: lib.mqc_adamw_step(rows(*v), count, *how, None, None)
    assert step(0, 64, 64, 64, 5, 0) == -1
    assert step(64, 64, 64, 64, -5, 0) == -2
    assert step(64, 64, 64, 64, 5, 9) == -3
    assert step(66, 64, 64, 64, 5, 0) == -4 and step(64, 64, 66, 64, 5, 0) == -4
    assert step(64, 65, 64, 64, 5, 1) == -4
    assert step(64, 64, 64, 64, 1 << 62, 0) == -5
    assert step(count=-1) == -2 and step(count=0) == 0
    assert step(0, 0, 0, 0, 0, 0) == 0  # nothing to do
    assert lib.mqc_adamw_step(None, 1, *how, None, None) == -1
    step8 = lambda *v: lib.mqc_adamw8_step(rows(*v), 1, *how, None, 1, None)
    assert step8(64, 64, 64, 64, 64, 0, 5, 0, 0) == -1
    assert step8(64, 64, 64, 64, 66, 64, 5, 0, 0) == -4
    assert step8(64, 64, 64, 64, 64, 64, 5, 4, 0) == -3
    assert lib.mqc_grad_norm_workspace_bytes(rows(64, 8193, 0, 64, 1, 1), 2) == 24
    assert lib.mqc_grad_norm_workspace_bytes(rows(64, -1, 0), 1) == -2
    fake = ctypes.c_void_p(4096)
    assert lib.mqc_grad_norm(rows(64, 10, 0), 1, 1.0, None, fake, fake, 64, None) == -1
    assert lib.mqc_grad_norm(rows(64, 10, 0), 1, 1.0, fake, fake, fake, 4, None) == -6


@pytest.mark.parametrize("copied", [copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))])
def test_copies_keep_their_settings(copied):
    p = torch.nn.Parameter(torch.ones(3))
    opt = copied(AdamW([p], lr=0.5, state_bits=8, min_8bit_size=2, max_norm=0.25, seed=11))
    assert (opt.min_8bit_size, opt.max_norm, opt.seed, opt.grad_norm) == (2, 0.25, 11, None)
    group, = opt.param_groups
    assert group["lr"] == 0.5 and group["state_bits"] == 8 and torch.equal(group["params"][0], p)
    group["params"][0].grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="ROCm device"):
        opt.step()


@pytest.mark.parametrize("copied", [copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))])
def test_copies_keep_8_bit_states(copied):
    p = torch.nn.Parameter(torch.ones(3))
    opt = AdamW([p], state_bits=8)
    codes = torch.tensor([1.0, -2.0, 0.5]).to(E4M3)
    opt.state[p] = {"step": 3, "exp_avg": codes, "exp_avg_scale": torch.tensor([0.5])}
    other = copied(opt)
    state = other.state[other.param_groups[0]["params"][0]]
    assert state["step"] == 3 and state["exp_avg"].dtype == E4M3
    assert torch.equal(state["exp_avg"].float(), codes.float()) and state["exp_avg_scale"].item() == 0.5
    assert state["exp_avg"].data_ptr() != codes.data_ptr()
    assert opt.state[p]["exp_avg"].dtype == E4M3
    new = torch.nn.Parameter(torch.ones(3))
    other.add_param_group({"params": [new]})
    assert other.state[new] == {}


def test_tensors_past_one_launch_are_refused():
    """2^32 threads and more along an axis, which HIP does not launch. (Without pointers: what is within
    the limit is refused for those.)"""
    lib, how = nat.load(), [1.0] * 8
    most = 4096 * ((1 << 24) - 1)
    for n, want in ((most, -1), (most + 1, -5)):
        assert lib.mqc_adamw_step(rows(0, 64, 64, 64, n, 0), 1, *how, None, None) == want
        assert lib.mqc_adamw8_step(rows(0, 64, 64, 64, 64, 64, n, 0, 0), 1, *how, None, 1, None) == want
        assert lib.mqc_grad_norm_workspace_bytes(rows(0, 2 * n, 0), 1) == want


def test_the_package_has_its_optimizer():
    """mambaqc_amd.optim.AdamW after `import mambaqc_amd` alone, as mambaqc_amd.kernels and .layers are."""
    code = "import mambaqc_amd; print(mambaqc_amd.optim.AdamW, mambaqc_amd.kernels, mambaqc_amd.layers)"
    root = Path(__file__).resolve().parents[1]
    subprocess.run([sys.executable, "-c", code], cwd=root, check=True)


@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64])
def test_states_do_not_follow_the_default_dtype(default):
    """A step under another default dtype refuses nothing but the CPU."""
    p, q = (torch.nn.Parameter(torch.ones(n, dtype=torch.float32)) for n in (600, 3))
    opt = AdamW([p, q], state_bits=8, min_8bit_size=100)
    before = torch.get_default_dtype()
    try:
        torch.set_default_dtype(default)
        p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
        with pytest.raises(RuntimeError, match="ROCm device"):
            opt.step()
    finally:
        torch.set_default_dtype(before)
    for s, names in ((opt.state[p], ("exp_avg_scale", "root_avg_sq_scale")),
                     (opt.state[q], ("exp_avg", "exp_avg_sq"))):
        assert not s or all(s[k].dtype == torch.float32 for k in names)
