"""The AdamW step (csrc/adamw.hip) against the formula in 64 bits: tensors of every type and odd size,
views, more than one table of them, clipping; the 8-bit states' codes, scales and means; the optimizer
against torch's.

Tolerances. In fp32, m and v are sums of two products: three roundings, at most 2^-22 of the terms'
absolute values. The update carries at most eight roundings (and the two means' own): 2^-20 of it. p
takes two more and half a step of its type.
"""
import copy
import math
import pickle

import pytest
import torch

import mambaqc_amd
from mambaqc_amd import _native as nat
from mambaqc_amd.optim import AdamW, adamw8_step_, adamw_step_, grad_norm, state_blocks

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn
HOW = {"lr": 3e-3, "betas": (0.9, 0.95), "eps": 1e-8, "weight_decay": 0.1}
# Elements: one to a few, around a lane's four, a block's 256, a workgroup's 4096, and none.
SIZES = [1, 2, 3, 4, 5, 255, 256, 257, 0, 1023, 4095, 4096, 4097, 8191, 20000]


def tensors(sizes, dtypes, seed=0, offset=0):
    """Parameters and gradients that start `offset` elements into their buffers."""
    gen = torch.Generator(DEV).manual_seed(seed)
    r = lambda n: torch.randn(n + offset, generator=gen, device=DEV)[offset:]
    ps = [r(n).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]
    if offset:
        ps = [torch.cat([p[:0].new_zeros(offset), p])[offset:] for p in ps]
    gs = [(10.0 ** -(i % 4) * r(n)).to(p.dtype) for i, (n, p) in enumerate(zip(sizes, ps))]
    ms = [0.1 * g.float() * r(n) for n, g in zip(sizes, gs)]
    vs = [(g.float() ** 2 + 1e-9) * r(n).abs() for n, g in zip(sizes, gs)]
    return ps, gs, ms, vs


def formula(p, g, m, v, step, clip=1.0, lr=None, betas=None, eps=None, weight_decay=None):
    p, g, m, v = (t.double() for t in (p, g, m, v))
    g = g * clip
    m, v = betas[0] * m + (1 - betas[0]) * g, betas[1] * v + (1 - betas[1]) * g * g
    update = lr * (m / (1 - betas[0] ** step)) / ((v / (1 - betas[1] ** step)).sqrt() + eps)
    return p * (1 - lr * weight_decay) - update, m, v, update


def hold_p(got, want, update, slack=2.0 ** -20):
    half = torch.finfo(got.dtype).eps / 2
    off = (got.double() - want).abs()
    assert (off <= (half + 2.0 ** -22) * want.abs() + slack * update.abs()
            + (2 ** -25 if got.dtype == torch.float16 else 1e-44)).all(), off.max()


@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], [torch.float16],
                                    [torch.bfloat16, torch.float32, torch.float16]])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("max_norm", [None, 0.5])
def test_step_32(dtypes, offset, max_norm):
    sizes = SIZES * 4  # 60 tensors: more than one table
    ps, gs, ms, vs = tensors(sizes, dtypes, offset=offset)
    old = [[t.clone() for t in ts] for ts in (ps, gs, ms, vs)]
    norm = adamw_step_(ps, gs, ms, vs, step=7, max_norm=max_norm, **HOW)
    total = math.sqrt(sum(g.double().square().sum().item() for g in gs))
    clip = 1.0
    if max_norm is None:
        assert norm is None
    else:
        assert abs(norm.item() - total) <= 2.0 ** -23 * total
        clip = min(1.0, max_norm / (total + 1e-6))
        assert clip < 1
    for i, p in enumerate(ps):
        p0, g0, m0, v0 = (ts[i] for ts in old)
        want, m, v, update = formula(p0, g0, m0, v0, 7, clip, **HOW)
        g = g0.double() * clip
        assert ((ms[i].double() - m).abs() <= 2.0 ** -22 * (0.9 * m0.abs() + 0.1 * g.abs())).all()
        assert ((vs[i].double() - v).abs() <= 2.0 ** -21 * v + 1e-44).all()
        # m's rounding, against the update of its terms rather than of their sum.
        spread = update.abs() * (0.9 * m0.abs() + 0.1 * g.abs()) / m.abs().clamp_min(1e-30)
        hold_p(p, want, update.abs() + spread)
        assert torch.equal(gs[i], g0)


def encoded(value):
    """A state's codes and scales, rounded to nearest."""
    n = value.numel()
    wide = torch.zeros(state_blocks(n) * 256, device=DEV)
    wide[:n] = value
    top = wide.view(-1, 256).abs().amax(1).clamp_min(2.0 ** -100)
    scale = torch.exp2(torch.ceil(torch.log2(top.double() / 448))).float()
    codes = (wide.view(-1, 256) / scale[:, None]).to(E4M3).view(-1)[:n]
    return codes.clone(), scale


def decoded(codes, scale):
    return codes.double() * scale.double().repeat_interleave(256)[:codes.numel()]


def neighbours(x):
    """The e4m3 numbers at or below and at or above |x| <= 448 (64 bits)."""
    x = x.abs()
    step = torch.exp2((torch.floor(torch.log2(x.clamp_min(2.0 ** -6)))) - 3)
    return (x / step).floor() * step, (x / step).ceil() * step


@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16, torch.float16]])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("max_norm", [None, 0.5])
def test_step_8(dtypes, offset, max_norm):
    sizes = SIZES * 4
    ps, gs, ms, vs = tensors(sizes, dtypes, offset=offset)
    m8, r8 = [encoded(m) for m in ms], [encoded(v.sqrt()) for v in vs]
    if offset:  # codes that start at odd bytes
        shift = lambda c: torch.cat([c.view(torch.uint8)[:0].new_zeros(1), c.view(torch.uint8)])[1:].view(E4M3)
        m8, r8 = ([(shift(c), s) for c, s in states] for states in (m8, r8))
    ms, rs = [decoded(*t) for t in m8], [decoded(*t) for t in r8]
    old = [p.clone() for p in ps]
    args = ([c for c, _ in m8], [s for _, s in m8], [c for c, _ in r8], [s for _, s in r8])
    norm = adamw8_step_(ps, gs, *args, step=7, seed=3, max_norm=max_norm, **HOW)
    total = math.sqrt(sum(g.double().square().sum().item() for g in gs))
    clip = 1.0 if max_norm is None else min(1.0, max_norm / (total + 1e-6))
    assert (norm is None) == (max_norm is None)
    for i, p in enumerate(ps):
        if p.numel() == 0:
            continue
        want, m, v, update = formula(old[i], gs[i], ms[i], rs[i] ** 2, 7, clip, **HOW)
        g = gs[i].double() * clip
        spread = update.abs() * (0.9 * ms[i].abs() + 0.1 * g.abs()) / m.abs().clamp_min(1e-30)
        hold_p(p, want, update.abs() + spread)
        for value, (code, scale) in ((m, m8[i]), (v.sqrt(), r8[i])):
            wide = torch.zeros(scale.numel() * 256, device=DEV, dtype=torch.float64)
            wide[:p.numel()] = value
            top = wide.view(-1, 256).abs().amax(1)
            assert (torch.frexp(scale)[0] == 0.5).all()  # a power of two
            assert (top <= 448 * scale.double() * (1 + 2.0 ** -20)).all()
            assert (top > 224 * scale.double() * (1 - 2.0 ** -20)).all()
            x = value / scale.double().repeat_interleave(256)[:p.numel()]
            low, high = neighbours(x * (1 - 2.0 ** -20))[0], neighbours(x * (1 + 2.0 ** -20))[1]
            got = code.double()
            assert ((got.abs() >= low) & (got.abs() <= high)).all()
            assert ((got == 0) | (got.sign() == value.sign())).all()
        assert (r8[i][0].double()[v > 0] > 0).all()


def test_rounding_keeps_the_means():
    """m's mean over seeds is m, and the mean of r^2 is v: each is off by at most 5 deviations of the
    mean of 4096 draws, one of which is at most half a step (of e4m3, 1/8 of the value; r^2: 17/64)."""
    n, draws = 256, 4096
    gen = torch.Generator(DEV).manual_seed(1)
    g = torch.exp(3 * torch.randn(n, generator=gen, device=DEV)) * 1e-3
    sums = [torch.zeros(n, device=DEV, dtype=torch.float64) for _ in range(2)]
    p, zero = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV, dtype=torch.uint8)
    for seed in range(draws):
        m, r = zero.clone().view(E4M3), zero.clone().view(E4M3)
        a, b = torch.ones(1, device=DEV), torch.ones(1, device=DEV)
        adamw8_step_([p], [g], [m], [a], [r], [b], step=5, seed=seed, **HOW)
        sums[0] += decoded(m, a)
        sums[1] += decoded(r, b) ** 2
    for got, want, scale, width in ((sums[0], 0.1 * g.double(), a, 1 / 16),
                                    (sums[1], 0.05 * g.double() ** 2, b, 17 / 128)):
        unit = scale.double() * 2.0 ** -9
        if width == 1 / 16:
            bound = 5 * torch.maximum(width * want, unit / 2) / math.sqrt(draws)
            assert ((got / draws - want).abs() <= bound + 1e-6 * want).all()
        else:
            normal = want.sqrt() >= 2.0 ** -6 * scale.double()  # below, steps are wider
            bound = 5 * width * want / math.sqrt(draws) + 1e-6 * want
            assert ((got / draws - want).abs() <= bound)[normal].all()
            # The smallest go to the least code that is not 0, never under.
            # Below 8 steps of 2^-9 a step of r^2 is at most 15 of its units, its deviation half that.
            assert ((got / draws) >= want - 37.5 * unit ** 2 / math.sqrt(draws))[~normal].all()


def test_small_updates_are_not_lost():
    """Gradients that drop to a tenth: v follows to a hundredth, though one update moves it by half a
    percent and a step of its codes is 12 to 25 % (rounding to nearest would leave it where it was)."""
    n = 4096
    betas, p = (0.9, 0.995), torch.zeros(4096, device=DEV)
    gen = torch.Generator(DEV).manual_seed(2)
    zero = lambda: torch.zeros(n, device=DEV, dtype=torch.uint8).view(E4M3)
    m, r, a, b = zero(), zero(), torch.ones(16, device=DEV), torch.ones(16, device=DEV)
    for step in range(1, 3001):
        size = 1.0 if step <= 1000 else 0.1
        g = size * torch.randn(n, generator=gen, device=DEV)
        adamw8_step_([p], [g], [m], [a], [r], [b], step=step, betas=betas, lr=0.0)
        if step == 1000:
            # E v = 1 - beta2^1000; sampling deviates by sqrt((1 - b) / (1 + b) 2 / n) = 1 %, rounding
            # by up to 30 % an element, 0.5 % of the mean: 5 % is five of both and more.
            assert abs((decoded(r, b) ** 2).mean().item() - (1 - 0.995 ** 1000)) < 0.05
    v = (decoded(r, b) ** 2).mean().item()
    left = 0.995 ** 2000
    assert abs(v - (0.01 * (1 - left) + left)) < 0.05 * 0.01


def test_nothing_but_nan_from_nan():
    """A NaN and an inf among gradients stay where they are: the others' states and scale are as
    without them."""
    n = 600
    ps, gs, ms, vs = tensors([n], [torch.float32])
    runs = []
    for bad in (False, True):
        p, g = ps[0].clone(), gs[0].clone()
        if bad:
            g[5], g[300] = float("nan"), float("inf")
        else:
            g[5] = g[300] = 0
        (m, a), (r, b) = encoded(ms[0]), encoded(vs[0].sqrt())
        adamw8_step_([p], [g], [m], [a], [r], [b], step=3, **HOW)
        runs.append((p, m, a, r, b))
    good = torch.ones(n, dtype=torch.bool, device=DEV)
    good[5] = good[300] = False
    (p0, m0, a0, r0, b0), (p1, m1, a1, r1, b1) = runs
    assert torch.equal(p0[good], p1[good]) and torch.equal(a0, a1) and torch.equal(b0, b1)
    for u, w in ((m0, m1), (r0, r1)):
        assert torch.equal(u.view(torch.uint8)[good], w.view(torch.uint8)[good])
        assert torch.isnan(w.float()[~good]).all()
    assert torch.isnan(p1[~good]).all()


def test_zero_gradients_and_states():
    n = 300
    p = torch.randn(n, device=DEV)
    p0, zero = p.clone(), torch.zeros(n, device=DEV, dtype=torch.uint8)
    m, r = zero.clone().view(E4M3), zero.clone().view(E4M3)
    a, b = torch.ones(2, device=DEV), torch.ones(2, device=DEV)
    adamw8_step_([p], [torch.zeros(n, device=DEV)], [m], [a], [r], [b], step=1, lr=0.1,
                 weight_decay=0.0)
    assert torch.equal(p, p0)
    assert (m.float() == 0).all() and (r.float() == 0).all()
    assert (a > 0).all() and torch.isfinite(a).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes", [[1], [3, 0, 8193], [70000, 5], [100] * 100])
def test_grad_norm(dtype, sizes):
    gs = [torch.randn(n, device=DEV).to(dtype) for n in sizes]
    want = math.sqrt(sum(g.double().square().sum().item() for g in gs))
    assert abs(grad_norm(gs).item() - want) <= 2.0 ** -23 * want
    odd = [torch.cat([g[:1], g])[1:] for g in gs]
    assert grad_norm(odd).item() == grad_norm(gs).item()


def test_grad_norm_of_large_and_bad_values():
    assert abs(grad_norm([torch.full((1000,), 1e30, device=DEV)]).item() / (1e30 * math.sqrt(1000)) - 1) < 1e-6
    assert abs(grad_norm([torch.full((1000,), 1e-30, device=DEV)]).item() / (1e-30 * math.sqrt(1000)) - 1) < 1e-6
    assert math.isnan(grad_norm([torch.tensor([1.0, float("nan")], device=DEV)]).item())
    assert math.isinf(grad_norm([torch.tensor([1.0, float("inf")], device=DEV)]).item())


def _models(dtype=torch.float32):
    torch.manual_seed(0)
    ref = torch.nn.Sequential(torch.nn.Linear(20, 300), torch.nn.Linear(300, 17)).double()
    ours = torch.nn.Sequential(torch.nn.Linear(20, 300), torch.nn.Linear(300, 17))
    ours.load_state_dict(ref.state_dict())
    return ref, ours.to(DEV, dtype)


def test_optimizer_against_torch():
    ref, ours = _models()
    groups = lambda m: [{"params": m[0].parameters(), "lr": 1e-2},
                        {"params": m[1].parameters(), "weight_decay": 0.3, "betas": (0.8, 0.9)}]
    a = torch.optim.AdamW(groups(ref), lr=1e-3)
    b = AdamW(groups(ours), lr=1e-3, max_norm=0.7)
    for step in range(12):
        gen = torch.Generator().manual_seed(step)
        for p, q in zip(ref.parameters(), ours.parameters()):
            p.grad = torch.randn(p.shape, generator=gen, dtype=torch.float64)
            q.grad = p.grad.float().to(DEV)
            p.grad = q.grad.double().cpu()
        if step in (3, 4):  # a parameter without a gradient keeps its own step count
            ref[1].bias.grad = ours[1].bias.grad = None
        norm = torch.nn.utils.clip_grad_norm_(ref.parameters(), 0.7)
        a.step()
        b.step()
        assert abs(b.grad_norm.item() - norm.item()) <= 2.0 ** -22 * norm.item()
    for p, q in zip(ref.parameters(), ours.parameters()):
        # Twelve steps of at most lr 1e-2 each, every one to 2^-19 of itself and 2^-23 of p.
        assert ((q.double().cpu() - p).abs() <= 12 * (2.0 ** -19 * 1e-2 + 2.0 ** -22 * p.abs())).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip(bits):
    _, model = _models(torch.bfloat16)
    _, other = _models(torch.bfloat16)
    first = AdamW(model.parameters(), lr=1e-2, state_bits=bits, seed=9)

    def go(opt, m, steps):
        for step in steps:
            gen = torch.Generator(DEV).manual_seed(step)
            for p in m.parameters():
                p.grad = torch.randn(p.shape, generator=gen, device=DEV).to(p.dtype)
            opt.step()

    go(first, model, range(3))
    saved = first.state_dict()
    kinds = {k: v.dtype for s in saved["state"].values() for k, v in s.items() if torch.is_tensor(v)}
    assert kinds["exp_avg"] in (torch.float32, E4M3)
    big = saved["state"][0]
    assert ("root_avg_sq" in big) == (bits == 8) and big["step"] == 3
    assert "exp_avg_sq" in saved["state"][1]  # the bias: too small for 8 bits
    other.load_state_dict(model.state_dict())
    second = AdamW(other.parameters(), lr=1e-2, state_bits=bits, seed=9)
    second.load_state_dict(saved)
    for s, t in zip(first.state.values(), second.state.values()):
        for k in s:
            assert (s[k] == t[k]) if k == "step" else (
                s[k].dtype == t[k].dtype and s[k].data_ptr() != t[k].data_ptr())
    go(first, model, range(3, 6))
    go(second, other, range(3, 6))
    for p, q in zip(model.parameters(), other.parameters()):
        assert torch.equal(p, q)


def test_copies_of_parameters_are_renewed():
    """The kernels write through pointers; what is kept of a 16-bit parameter in fp32 has to follow."""
    p = torch.nn.Parameter(torch.randn(64, device=DEV).bfloat16())
    before, version = nat.param_f32(p).clone(), p._version
    p.grad = torch.ones_like(p)
    AdamW([p], lr=0.5).step()
    assert p._version > version
    assert torch.equal(nat.param_f32(p), p.detach().float())
    assert not torch.equal(nat.param_f32(p), before)
    # And autograd refuses a backward over a parameter that was changed in between.
    w = torch.nn.Parameter(torch.ones(4, device=DEV))
    loss = (w * w).sum()
    w.grad = torch.ones_like(w)
    AdamW([w]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


def test_refusals():
    p = torch.nn.Parameter(torch.ones(8, 4, device=DEV))
    p.grad = torch.ones_like(p)
    opt = AdamW([p])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="not captured"):
        with torch.cuda.graph(graph):
            opt.step()
    torch.cuda.synchronize()
    flat = [torch.ones(32, device=DEV) for _ in range(4)]
    with pytest.raises(ValueError, match="contiguous"):
        adamw_step_([torch.ones(8, 4, device=DEV).T], [torch.ones(4, 8, device=DEV)], [flat[0]],
                    [flat[1]], step=1)
    with pytest.raises(RuntimeError, match="ROCm device"):
        adamw_step_([flat[0]], [torch.ones(32)], [flat[1]], [flat[2]], step=1)


def test_same_bits_again_and_on_another_stream():
    sizes = [5000, 300, 70001]
    runs = []
    for stream in (None, torch.cuda.Stream()):
        ps, gs, ms, vs = tensors(sizes, [torch.bfloat16], seed=4)
        m8, r8 = [encoded(m) for m in ms], [encoded(v.sqrt()) for v in vs]
        args = ([c for c, _ in m8], [s for _, s in m8], [c for c, _ in r8], [s for _, s in r8])
        torch.cuda.synchronize()
        if stream is None:
            norm = adamw8_step_(ps, gs, *args, step=2, seed=5, max_norm=1.0, **HOW)
        else:
            with torch.cuda.stream(stream):
                norm = adamw8_step_(ps, gs, *args, step=2, seed=5, max_norm=1.0, **HOW)
        torch.cuda.synchronize()
        runs.append([norm, *ps, *(t.view(torch.uint8) for t in args[0] + args[2]), *args[1], *args[3]])
    for u, v in zip(*runs):
        assert torch.equal(u, v)


@pytest.mark.parametrize("bits", [32, 8])
def test_block_trains(bits):
    """A few steps of the framework's block: the loss on one batch goes down."""
    torch.manual_seed(0)
    block = mambaqc_amd.QuaternionMamba2Block(32, d_state=4).to(DEV)
    x, want = torch.randn(2, 20, 32, device=DEV), torch.randn(2, 20, 32, device=DEV)
    opt = AdamW(block.parameters(), lr=3e-3, state_bits=bits, min_8bit_size=256, max_norm=1.0)
    losses = []
    for _ in range(30):
        opt.zero_grad()
        loss = (block(x) - want).square().mean()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    assert losses[-1] < 0.9 * losses[0]


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(bits):
    """More tensors than one launch's table, of the step (88, with 8-bit states 60) and the norm (160)."""
    sizes = [3 + 7 * i for i in range(200)]
    ps, gs, ms, vs = tensors(sizes, [torch.float32, torch.bfloat16])
    old = [p.clone() for p in ps]
    if bits == 32:
        norm = adamw_step_(ps, gs, [m.clone() for m in ms], [v.clone() for v in vs], step=7,
                           max_norm=0.5, **HOW)
    else:
        m8, r8 = [encoded(m) for m in ms], [encoded(v.sqrt()) for v in vs]
        ms, vs = [decoded(*t) for t in m8], [decoded(*t) ** 2 for t in r8]
        norm = adamw8_step_(ps, gs, [c for c, _ in m8], [s for _, s in m8], [c for c, _ in r8],
                            [s for _, s in r8], step=7, max_norm=0.5, **HOW)
    total = math.sqrt(sum(g.double().square().sum().item() for g in gs))
    assert abs(norm.item() - total) <= 2.0 ** -23 * total
    clip = min(1.0, 0.5 / (total + 1e-6))
    for p, p0, g, m, v in zip(ps, old, gs, ms, vs):
        want, m1, _, update = formula(p0, g, m, v, 7, clip, **HOW)
        spread = update.abs() * (0.9 * m.abs() + 0.1 * g.abs() * clip) / m1.abs().clamp_min(1e-30)
        hold_p(p, want, update.abs() + spread)


def test_more_than_the_caches_hold():
    """States and parameters stored past the caches (over 256 MiB in all)."""
    ps, gs, ms, vs = tensors([17_000_003], [torch.float32])
    want, m, v, update = formula(ps[0], gs[0], ms[0], vs[0], 7, **HOW)
    spread = update.abs() * (0.9 * ms[0].abs() + 0.1 * gs[0].abs()) / m.abs().clamp_min(1e-30)
    adamw_step_(ps, gs, ms, vs, step=7, **HOW)
    hold_p(ps[0], want, update.abs() + spread)
    assert ((vs[0].double() - v).abs() <= 2.0 ** -21 * v + 1e-44).all()


@pytest.mark.parametrize("scale", [1e-25, 1e-12, 1.0, 1e12, 1e18])
def test_8_bit_states_of_any_size(scale):
    """Values at which a square underflows or overflows, beside ordinary blocks: the same codes as the
    formula's neighbours, and parameters that follow it."""
    n = 1024
    gen = torch.Generator(DEV).manual_seed(3)
    g = torch.randn(n, generator=gen, device=DEV)
    g[256:512] *= scale
    p = torch.zeros(n, device=DEV)
    (m, a), (r, b) = encoded(torch.zeros(n, device=DEV)), encoded(torch.zeros(n, device=DEV))
    adamw8_step_([p], [g], [m], [a], [r], [b], step=1, lr=1e-2, betas=(0.9, 0.95), weight_decay=0.0)
    g64 = g.double()
    for value, code, sc in ((0.1 * g64, m, a), ((0.05 * (g * g).double()).sqrt(), r, b)):
        x = value / sc.double().repeat_interleave(256)
        low, high = neighbours(x * (1 - 2.0 ** -20))[0], neighbours(x * (1 + 2.0 ** -20))[1]
        got = code.double()
        assert ((got.abs() >= low) & (got.abs() <= high) | (got == 2.0 ** -9) & (x > 0)).all()
    big = (g * g) >= 2.0 ** -120
    step = 1e-2 * g64 / (((g * g).double()).sqrt() + 1e-8)
    assert ((p.double() + step).abs() <= 2.0 ** -18 * 1e-2)[big].all()
    assert p.isfinite().all()


@pytest.mark.parametrize("bits", [32, 8])
def test_offsets_past_32_bits(bits):
    """Elements more than 2^31 into a tensor, its states' among them."""
    n = 2 ** 31 + 1025
    p = torch.zeros(n, device=DEV, dtype=torch.bfloat16)
    g = torch.zeros_like(p)
    at = torch.tensor([0, 2 ** 31 - 1, 2 ** 31, 2 ** 31 + 700, n - 1], device=DEV)
    g[at] = 0.25
    how = {"step": 1, "lr": 0.5, "betas": (0.9, 0.95), "weight_decay": 0.0}
    if bits == 32:
        m, v = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
        adamw_step_([p], [g], [m], [v], **how)
        assert ((m[at] - 0.025).abs() < 1e-8).all() and int((m != 0).sum()) == 5
    else:
        c = [torch.zeros(n, device=DEV, dtype=torch.uint8).view(E4M3) for _ in range(2)]
        s = [torch.ones(state_blocks(n), device=DEV) for _ in range(2)]
        adamw8_step_([p], [g], [c[0]], [s[0]], [c[1]], [s[1]], **how)
        for code, scale, want in ((c[0], s[0], 0.025), (c[1], s[1], 0.25 * 0.05 ** 0.5)):
            got = code.view(torch.uint8)[at].view(E4M3).float() * scale[at // 256]
            assert ((got - want).abs() <= want / 8).all()
            assert int((code.view(torch.uint8) != 0).sum()) == 5
    assert (p[at] == -0.5).all() and int((p != 0).sum()) == 5
    assert abs(grad_norm([g]).item() - 0.25 * 5 ** 0.5) < 1e-6


def test_8_bit_seeds_of_any_size():
    """Seeds count modulo 2^32, those past 64 bits and negative ones among them."""
    n = 1000
    results = []
    for seed in (7, 7 + (1 << 32), 7 + (5 << 64), 7 - (1 << 32)):
        gen = torch.Generator(DEV).manual_seed(6)
        ps, gs = [[torch.randn(n, generator=gen, device=DEV) for _ in range(2)] for _ in range(2)]
        codes = [[torch.zeros(n, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn)
                  for _ in range(2)] for _ in range(2)]
        scales = [[torch.ones(state_blocks(n), device=DEV) for _ in range(2)] for _ in range(2)]
        adamw8_step_(ps, gs, codes[0], scales[0], codes[1], scales[1], step=1, seed=seed)
        results.append([t.view(torch.uint8) for t in (*ps, *codes[0], *codes[1])])
    for got in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got, results[0]))


def test_a_step_past_the_cache_equals_its_parts():
    """Parameters and states past 256 MiB in one call: the same bits as tensor by tensor."""
    sizes = [9_000_001, 4097, 8_500_003, 0, 5]
    gen = torch.Generator(DEV).manual_seed(7)
    lists = [[torch.randn(n, generator=gen, device=DEV) for n in sizes] for _ in range(4)]
    lists[3] = [v.abs() for v in lists[3]]
    apart = [[t.clone() for t in one] for one in lists]
    adamw_step_(*lists, step=4, lr=1e-2)
    for i in range(len(sizes)):
        adamw_step_(*([one[i]] for one in apart), step=4, lr=1e-2)
    for got, want in zip(lists, apart):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_negated_gradients():
    """A gradient that torch negates as it reads it (the imaginary part of a conjugate)."""
    p = torch.nn.Parameter(torch.ones(5, 1, device=DEV))
    q = torch.nn.Parameter(torch.ones(5, 1, device=DEV))
    p.grad = torch.ones(5, 1, device=DEV) * torch.arange(5, device=DEV)[:, None]
    q.grad = torch._neg_view(-p.grad)
    assert q.grad.is_neg()
    AdamW([p], lr=0.1).step()
    AdamW([q], lr=0.1).step()
    assert torch.equal(p, q)
    with pytest.raises(ValueError, match="do not take"):
        adamw_step_([torch._neg_view(torch.ones(5, device=DEV))], [torch.ones(5, device=DEV)],
                    [torch.zeros(5, device=DEV)], [torch.zeros(5, device=DEV)], step=1)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("copied", [copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))])
def test_copies_go_on_with_the_same_bits(copied, bits):
    gen = torch.Generator(DEV).manual_seed(3)
    params = [torch.nn.Parameter(torch.randn(n, generator=gen, device=DEV)) for n in (5000, 300)]
    opt = AdamW(params, lr=0.1, state_bits=bits, min_8bit_size=1000, max_norm=0.5, seed=5)

    def step(params, opt, seed):
        gen = torch.Generator(DEV).manual_seed(seed)
        for p in params:
            p.grad = torch.randn(p.shape, generator=gen, device=DEV)
        opt.step()

    step(params, opt, 1)
    other, twins = copied((opt, params))
    for seed in (2, 3):
        step(params, opt, seed)
        step(twins, other, seed)
        for p, q in zip(params, twins):
            assert p is not q and torch.equal(p, q)
        assert torch.equal(opt.grad_norm, other.grad_norm)


@pytest.mark.parametrize("bits", [8, 32])
def test_parameters_that_share_memory_are_refused(bits):
    """Two workgroups would write one parameter side by side; neighbours in one buffer are fine."""
    flat = torch.ones(3000, device=DEV)
    new = lambda n: torch.zeros(n, device=DEV)
    code = lambda n: torch.zeros(n, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)

    def step(params):
        ns, grads = [p.numel() for p in params], [torch.ones_like(p) for p in params]
        if bits == 32:
            return adamw_step_(params, grads, [new(n) for n in ns], [new(n) for n in ns], step=1)
        scales = lambda: [torch.ones(state_blocks(n), device=DEV) for n in ns]
        return adamw8_step_(params, grads, [code(n) for n in ns], scales(), [code(n) for n in ns], scales(),
                            step=1)

    for bad in ([flat[:10], flat[:10]], [flat[100:700], flat[:101]], [flat[:3000], flat[50:60], new(4)]):
        with pytest.raises(ValueError, match="share memory"):
            step(bad)
    assert (flat == 1).all()
    step([flat[1000:2000], flat[:1000], flat[2000:], flat[500:500]])
    assert (flat < 1).all()
    p = torch.nn.Parameter(new(5000))
    p.grad = torch.ones_like(p)
    with pytest.warns(UserWarning, match="duplicate parameters"):
        opt = AdamW([p, p], state_bits=bits)
    with pytest.raises(ValueError, match="share memory"):
        opt.step()
