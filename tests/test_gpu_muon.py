"""orthogonalize and the Muon step (csrc/ortho.hip) against the iteration in 64 bits: sides of one to past
the tiles, tall and wide, stacks, lists of many shapes and types, weak directions, zero matrices, streams and
graphs, and the optimizer.

Tolerances, of the 2-norm of the difference over the result's. fp32 and fp16: a product's pieces leave out
2^-22 of each value and an accumulator rounds at 2^-24 per 32 products, as squares 2^-21 a product; fifteen
products, and weak directions' share of a rounding grows with them and no faster: 2^-21 sqrt(15) 2 = 2^-18.
bf16, from shorter sides of 256 on: operands of 11 bits are off by 2^-12 / sqrt(3) as squares, ten of them a
result of which each step keeps at most its own size: 2^-12 sqrt(10 / 3) = 4.5e-4, and 2 for A^2, whose two
roundings are one: the bound is 2^-9 (below, pairs: fp32's). Half a step of the type comes on top (as squares its uniform share, 1 / sqrt(3)).
"""
import copy

import pytest
import torch

from mambaqc_amd.optim import COEFFICIENTS, Muon, muon_step_, orthogonalize

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
REL = {torch.float32: 2.0 ** -18, torch.float16: 2.0 ** -18, torch.bfloat16: 2.0 ** -9}


def iterate(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = x.double()
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp_min(eps)
    for _ in range(steps):
        if x.shape[-2] <= x.shape[-1]:
            g = x @ x.mT
            x = a * x + (b * g + c * (g @ g)) @ x
        else:
            g = x.mT @ x
            x = a * x + x @ (b * g + c * (g @ g))
    return x


def hold(what, got, want, rel):
    off = (got.double() - want).flatten(0, -3).flatten(1) if got.dim() > 2 else (got.double() - want).reshape(1, -1)
    size = want.reshape(off.shape).norm(dim=1)
    half = torch.finfo(got.dtype).eps / 2
    assert got.shape == want.shape, what
    assert (off.norm(dim=1) <= (rel + half) * size + 1e-30).all(), (what, off.norm(dim=1) / size, rel)


def make(shape, dtype, seed=0, kind="normal"):
    gen = torch.Generator(DEV).manual_seed(seed + sum(shape))
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    if kind == "weak":  # a few strong directions over noise of a thousandth
        return (r(*shape[:-1], 4) @ r(*shape[:-2], 4, shape[-1]) + 1e-3 * r(*shape)).to(dtype)
    return r(*shape).to(dtype)


SHAPES = [(1, 1), (1, 7), (5, 1), (2, 3), (16, 16), (17, 40), (3, 33, 70), (63, 64), (64, 65), (2, 130, 129),
          (128, 256), (300, 70), (5, 2, 20, 31), (515, 1000), (1030, 260), (70000, 8), (24, 1100, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(dtype, shape):
    x = make(shape, dtype)
    y = orthogonalize(x)
    assert y.dtype == dtype and y.shape == x.shape
    hold("x", y, iterate(x), REL[dtype])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(200, 300), (600, 128), (12, 700, 500)])
def test_weak_directions(dtype, shape):
    """They grow 3.44 times a step, 485 in all, and a rounding of the whole with them, against a result of
    about the strong directions' norm, 1.4 and more: pieces hold X_0 to 2^-23 of a norm of 1, and the products
    of each step (A's pieces and A^2's) to 2^-22.5, of which four steps, three, .. make 141, 41, .. times as
    much: as squares 2^-23 (485^2 + 2 (141^2 + 41^2 + 12^2))^1/2 / 1.4 = 2^-23 377; twice that is allowed."""
    x = make(shape, dtype, kind="weak")
    hold("x", orthogonalize(x), iterate(x), REL[dtype] + 2 * 377 * 2.0 ** -23)


@pytest.mark.parametrize("steps,coefficients", [(1, COEFFICIENTS), (2, COEFFICIENTS), (12, (1.875, -1.25, 0.375)),
                                                (6, (1.5, -0.5, 0.0))])
def test_steps_and_coefficients(steps, coefficients):
    x = make((90, 200), torch.float32)
    y = orthogonalize(x, steps=steps, coefficients=coefficients)
    hold("x", y, iterate(x, steps, coefficients), REL[torch.float32] * max(1, steps / 5))


def test_sizes_of_values():
    """The norm is divided out, whatever it is; below eps it is eps; zeros stay zeros."""
    x = make((40, 90), torch.float32)
    y = orthogonalize(x)
    for size in (1e-30, 1e-20, 1e15, 1e30):
        hold(size, orthogonalize(x * size, eps=0.0), y.double(), REL[torch.float32])
    small = x / x.norm() * 1e-9
    hold("eps", orthogonalize(small), iterate(small), REL[torch.float32])
    assert (orthogonalize(torch.zeros(3, 20, 30, device=DEV)) == 0).all()
    stack = make((3, 20, 30), torch.float32)
    clean = orthogonalize(stack)
    stack[1, 3, 4] = float("nan")
    got = orthogonalize(stack)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[2], clean[2]) and got[1].isnan().any()


def test_views_and_empty():
    x = make((2, 60, 50), torch.float32)
    assert torch.equal(orthogonalize(x.mT.contiguous().mT), orthogonalize(x))
    wide = make((2, 60, 100), torch.bfloat16)
    assert torch.equal(orthogonalize(wide[..., 3:53]), orthogonalize(wide[..., 3:53].contiguous()))
    odd = torch.cat([torch.zeros(1, device=DEV), x.reshape(-1)])[1:].view(2, 60, 50)
    assert torch.equal(orthogonalize(odd), orthogonalize(x))
    for shape in ((0, 5), (5, 0), (0, 3, 4)):
        assert orthogonalize(torch.empty(shape, device=DEV)).shape == shape


def reference(p, g, m, lr, mu, nesterov, decay, **how):
    m = mu * m.double() + (1 - mu) * g.double()
    u = mu * m + (1 - mu) * g.double() if nesterov else m
    size = max(1, p.shape[0] / p.shape[1]) ** 0.5
    return p.double() * (1 - lr * decay) - lr * size * iterate(u, **how), m


# Every shape twice and more than one launch's shapes and matrices.
LIST = [(64, 256), (128, 128), (256, 64), (30, 31), (1, 9), (7, 1)] * 3 + [(20 + i, 40) for i in range(20)]


@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], TYPES])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step(dtypes, nesterov):
    lr, mu, decay = 0.05, 0.9, 0.2
    types = [dtypes[i % len(dtypes)] for i in range(len(LIST))]
    params = [make(s, t, seed=i) * 0.02 for i, (s, t) in enumerate(zip(LIST, types))]
    grads = [make(s, t, seed=100 + i) for i, (s, t) in enumerate(zip(LIST, types))]
    momenta = [make(s, torch.float32, seed=200 + i) for i, s in enumerate(LIST)]
    for _ in range(2):
        want = [reference(p, g, m, lr, mu, nesterov, decay) for p, g, m in zip(params, grads, momenta)]
        versions = [p._version for p in params]
        assert muon_step_(params, grads, momenta, lr=lr, momentum=mu, nesterov=nesterov,
                          weight_decay=decay) is None
        assert all(p._version > v for p, v in zip(params, versions))
        for i, (p, m, (wp, wm), t) in enumerate(zip(params, momenta, want, types)):
            hold(("m", i), m, wm, 2.0 ** -21)
            # The update is as large as the parameter and more here: its error counts whole, times the
            # update's share.
            update = wp.norm() + lr * max(1, p.shape[0] / p.shape[1]) ** 0.5 * min(p.shape) ** 0.5
            off = (p.double() - wp).norm()
            assert off <= (REL[t] + 2.0 ** -20) * update + torch.finfo(t).eps / 2 * wp.norm(), (i, off / update)


def test_many_matrices_of_one_shape():
    params = [make((20, 24), torch.float32, seed=i) for i in range(150)]
    grads = [make((20, 24), torch.float32, seed=1000 + i) for i in range(150)]
    momenta = [torch.zeros(20, 24, device=DEV) for _ in range(150)]
    want = [reference(p, g, m, 0.1, 0.95, True, 0.0)[0] for p, g, m in zip(params, grads, momenta)]
    muon_step_(params, grads, momenta, lr=0.1, weight_decay=0.0)
    for i, (p, w) in enumerate(zip(params, want)):
        hold(i, p, w, REL[torch.float32])
    muon_step_([], [], [])
    muon_step_([torch.empty(0, 4, device=DEV)], [torch.empty(0, 4, device=DEV)], [torch.empty(0, 4, device=DEV)])


def test_optimizer():
    """Two groups, a matrix without a gradient, bf16 parameters; state dicts, copies and loading go on
    with the same bits."""
    def model():
        ps = [torch.nn.Parameter(make(s, t, seed=i)) for i, (s, t) in
              enumerate([((30, 50), torch.float32), ((64, 20), torch.bfloat16), ((30, 50), torch.float32),
                         ((9, 9), torch.float32)])]
        return ps, Muon([{"params": ps[:2]}, {"params": ps[2:], "lr": 0.01, "nesterov": False}], lr=0.02)

    def steps(ps, opt, first, count):
        for i in range(first, first + count):
            for j, p in enumerate(ps[:3]):
                p.grad = make(p.shape, p.dtype, seed=50 + 10 * i + j)
            opt.step()

    ps, opt = model()
    want = [p.detach().double().clone() for p in ps]
    ms = [torch.zeros_like(w) for w in want]
    steps(ps, opt, 0, 1)
    for j in range(3):
        lr, nesterov = (0.02, True) if j < 2 else (0.01, False)
        g = make(ps[j].shape, ps[j].dtype, seed=50 + j)
        w, m = reference(want[j], g, ms[j], lr, 0.95, nesterov, 0.1)
        hold(j, ps[j].detach(), w, REL[ps[j].dtype])
        assert opt.state[ps[j]]["momentum_buffer"].dtype == torch.float32
        hold(j, opt.state[ps[j]]["momentum_buffer"], m, 2.0 ** -21)
    assert torch.equal(ps[3].detach().double(), want[3]) and ps[3] not in opt.state
    saved, held = copy.deepcopy(opt.state_dict()), [p.detach().clone() for p in ps]
    steps(ps, opt, 1, 2)
    qs, other = model()
    with torch.no_grad():
        for q, h in zip(qs, held):
            q.copy_(h)
    other.load_state_dict(saved)
    steps(qs, other, 1, 2)
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
    assert opt.step(lambda: 3.0) == 3.0


def test_learns():
    """A step runs and moves every parameter; how far a loss falls is no matter."""
    w = torch.nn.Parameter(make((40, 30), torch.float32))
    opt = Muon([w], lr=0.1)
    before = w.detach().clone()
    (w.square().sum()).backward()
    opt.step()
    assert (w.detach() != before).any() and w.isfinite().all()
    opt.zero_grad()
    opt.step()


def test_repeats_streams_and_graphs():
    x = make((6, 200, 330), torch.bfloat16)
    params, grads = [make((70, 90), torch.float32)], [make((70, 90), torch.float32, seed=1)]
    momenta = [torch.zeros(70, 90, device=DEV)]
    first = orthogonalize(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = orthogonalize(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, other)
    start = [params[0].clone(), momenta[0].clone()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = orthogonalize(x)
        muon_step_(params, grads, momenta)
    for rep in range(4):
        x.copy_(make(x.shape, torch.bfloat16, seed=rep))
        params[0].copy_(start[0])
        momenta[0].copy_(start[1])
        graph.replay()
        torch.cuda.synchronize()
        got = [out.clone(), params[0].clone(), momenta[0].clone()]
        params[0].copy_(start[0])
        momenta[0].copy_(start[1])
        muon_step_(params, grads, momenta)
        for u, v in zip(got, [orthogonalize(x), params[0], momenta[0]]):
            assert torch.equal(u, v), rep


def test_refusals():
    p = make((4, 5), torch.float32)
    with pytest.raises(ValueError, match="share memory"):
        muon_step_([p, p], [p.clone(), p.clone()], [p.clone(), p.clone()])
    with pytest.raises(ValueError, match="share memory"):
        muon_step_([p], [p.clone()], [p])
    opt = Muon([torch.nn.Parameter(p), torch.nn.Parameter(p)])
    for q in opt.param_groups[0]["params"]:
        q.grad = p.clone()
    with pytest.raises(ValueError, match="share memory"):
        opt.step()
    with pytest.raises(ValueError, match="contiguous"):
        muon_step_([p.T], [p.T.clone()], [p.T.contiguous()])
    with pytest.raises(RuntimeError, match="ROCm device"):
        muon_step_([p], [p.cpu()], [p.clone()])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(16, 900, 1030), (17, 1030, 770), (300, 5000), (3, 2500, 130)])
def test_large_tiles_and_shared_sides(dtype, shape):
    """Last products of 256 tiles of 256 by 256 and more, odd ones; first products shared along the long side."""
    x = make(shape, dtype)
    hold("x", orthogonalize(x), iterate(x), REL[dtype])


@pytest.mark.parametrize("dtype", TYPES)
def test_muon_step_of_large_tiles_in_a_graph(dtype):
    """Tall and wide ones beside small ones and a long one; captured as the first such call of a process too."""
    shapes = [(1000, 900)] * 9 + [(520, 2100)] * 6 + [(64, 40), (70, 4500)]
    params = [make(s, dtype, seed=i) for i, s in enumerate(shapes)]
    grads = [make(s, dtype, seed=100 + i) for i, s in enumerate(shapes)]
    momenta = [torch.zeros(s, device=DEV) for s in shapes]
    before = [p.clone() for p in params]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon_step_(params, grads, momenta, lr=0.5, momentum=0.9, weight_decay=0.1)
    for rep in range(3):
        for p, b, m in zip(params, before, momenta):
            p.copy_(b), m.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = [p.clone() for p in params]
        for p, b, m in zip(params, before, momenta):
            p.copy_(b), m.zero_()
        muon_step_(params, grads, momenta, lr=0.5, momentum=0.9, weight_decay=0.1)
        assert all(torch.equal(u, p) for u, p in zip(got, params))
    for p, b, g, s in zip(params, before, grads, shapes):
        # m = 0.1 g, u = 0.9 m + 0.1 g: a multiple of g.
        step = 0.5 * max(1.0, s[0] / s[1]) ** 0.5 * iterate(g)
        hold("p", p, b.double() * (1 - 0.5 * 0.1) - step, REL[dtype])


@pytest.mark.parametrize("size", [1e-38, 1e-37, 1e36, 1e37])
@pytest.mark.parametrize("shape", [(40, 90), (90, 40), (300, 280)])
def test_norms_past_the_ends_of_fp32(size, shape):
    """Norms that no fp32 number holds, and ones whose inverse is none."""
    x = make(shape, torch.float32) * size
    assert x.isfinite().all()
    hold("x", orthogonalize(x, eps=0.0), iterate(x, eps=0.0), REL[torch.float32])
    p, m = make(shape, torch.float32), torch.zeros(shape, device=DEV)
    want, _ = reference(p, x, m, 0.5, 0.0, False, 0.0, eps=0.0)
    muon_step_([p], [x], [m], lr=0.5, momentum=0.0, nesterov=False, weight_decay=0.0, eps=0.0)
    hold("p", p, want, REL[torch.float32])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (20, 33), (300, 280)])
def test_values_just_below_what_the_iteration_holds(dtype, shape):
    """Elements of X, A and b A + c A^2 have to be below 255. One direction, whose singular value goes 1 -> 15.9 ->
    52.6, with A = 252.8 in the second step; and one with b A + c A^2 = 253 and X = 254."""
    x = make((shape[0], 1), torch.float32) @ make((1, shape[1]), torch.float32, seed=5)
    x = (x / x.abs().max()).to(dtype)
    if dtype != torch.float32 and shape != (1, 1):  # (rounded, it has more directions than one)
        x = torch.zeros_like(x)
        x[3, 5] = -1.0
    for coefficients in ((15.95, -0.05, 0.0), (1.0, 13.0, 240.0)):
        steps = 1 if coefficients[0] == 1.0 else 2
        want = iterate(x, steps, coefficients)
        assert want.isfinite().all()
        hold(coefficients, orthogonalize(x, steps=steps, coefficients=coefficients), want, REL[dtype])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(2048, 2048), (2, 2100, 3000), (2500, 2200)])
def test_long_short_sides(dtype, shape):
    x = make(shape, dtype)
    hold("x", orthogonalize(x), iterate(x), REL[dtype])


@pytest.mark.parametrize("dtype", TYPES)
def test_short_sides_past_8192(dtype):
    """All three products sum over n = 8500 elements, for which the fp32 accumulators count too: three roundings
    per 32 elements, each 2^-24 / sqrt(3) (as squares) of a partial sum that is 1 / sqrt(2) of the whole one on
    the average, (3 n / 32)^1/2 2^-24 / sqrt(6) = 2^-20.5 a product beside the 2^-21 above. Of fifteen products,
    twice that: 2^-17.2."""
    x = make((8500, 8400), dtype)
    rel = 2 * 15 ** 0.5 * (2.0 ** -42 + 3 * 8500 / 32 * 2.0 ** -48 / 6) ** 0.5
    hold("x", orthogonalize(x), iterate(x), rel)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps_go_downhill(dtype):
    """Of |w - target|^2 / 2 the update X of the gradient has <X, gradient> above 0.6 of its singular values'
    sum (the iteration ends between 0.68 and 1.21): with steps of at most a tenth of the least singular value
    of w - target the loss falls in each."""
    target = torch.eye(30, 40, device=DEV) * 3
    w = torch.nn.Parameter(torch.zeros(30, 40, device=DEV, dtype=dtype))
    opt = Muon([w], lr=0.1, momentum=0.0, weight_decay=0.0)
    losses = []
    for _ in range(6):
        loss = (w.float() - target).square().sum() / 2
        losses.append(loss.item())
        opt.zero_grad()
        loss.backward()
        opt.step()
    assert all(b < a for a, b in zip(losses, losses[1:])), losses


def rounded_once(what, got, want, rel):
    """Each element is want's rounding, but for an error before it of rel as a 2-norm, of which one of up to a
    million elements has eight times the root mean square at most."""
    off, rms = (got.double() - want).abs(), want.square().mean().sqrt()
    bad = ~(off <= torch.finfo(got.dtype).eps / 2 * want.abs() + 8 * rel * rms)
    assert not bad.any(), (what, int(bad.sum()), (off / rms)[bad][:4], (want / rms)[bad][:4])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(300, 280), (2, 515, 1000), (700, 260), (256, 256), (40, 600)])
def test_rounded_once(dtype, shape):
    """16-bit matrices too are iterated at fp32's accuracy: their only rounding to 16 bits is the last."""
    x = make(shape, dtype)
    rounded_once("x", orthogonalize(x), iterate(x), 2.0 ** -18)


@pytest.mark.parametrize("dtype", TYPES)
def test_muon_step_rounds_once(dtype):
    shapes = [(300, 280), (256, 512), (40, 30), (515, 300)]
    params = [0.02 * make(s, dtype, seed=i) for i, s in enumerate(shapes)]
    grads = [make(s, dtype, seed=100 + i) for i, s in enumerate(shapes)]
    momenta = [make(s, torch.float32, seed=200 + i) for i, s in enumerate(shapes)]
    want = [reference(p, g, m, 0.02, 0.95, True, 0.1) for p, g, m in zip(params, grads, momenta)]
    opt = Muon([torch.nn.Parameter(p.clone()) for p in params], lr=0.02)
    muon_step_(params, grads, momenta, lr=0.02)
    for i, (p, (w, _)) in enumerate(zip(params, want)):
        rounded_once(i, p, w, 2.0 ** -18)
    for p, g in zip(opt.param_groups[0]["params"], grads):
        before, p.grad = p.detach().clone(), g
        opt.step()
        rounded_once("opt", p.detach(), reference(before, g, 0 * g, 0.02, 0.95, True, 0.1)[0], 2.0 ** -18)
        p.grad = None


@pytest.mark.parametrize("kind", ["normal", "weak"])
@pytest.mark.parametrize("shape", [(300, 280), (5, 600, 300), (256, 2100), (900, 1030)])
def test_fast_bf16(shape, kind):
    """Operands of 11 bits (the tolerance above)."""
    x = make(shape, torch.bfloat16, kind=kind)
    y = orthogonalize(x, fast_bf16=True)
    rel = 2.0 ** -9 + (2 * 377 * 2.0 ** -23 if kind == "weak" else 0)
    hold("x", y, iterate(x), rel)
    assert not torch.equal(y, orthogonalize(x))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(300, 280), (255, 400), (30, 20)])
def test_fast_bf16_leaves_others_as_they_are(dtype, shape):
    x = make(shape, dtype)
    same = torch.equal(orthogonalize(x, fast_bf16=True), orthogonalize(x))
    assert same == (dtype != torch.bfloat16 or min(shape) < 256)


def test_fast_bf16_steps():
    """In a list beside other types and sizes, in an optimizer's group and in a graph."""
    shapes = [(300, 280), (64, 40), (300, 280), (280, 512), (300, 280)]
    types = [torch.bfloat16, torch.bfloat16, torch.float32, torch.bfloat16, torch.float16]
    params = [0.02 * make(s, t, seed=i) for i, (s, t) in enumerate(zip(shapes, types))]
    grads = [make(s, t, seed=100 + i) for i, (s, t) in enumerate(zip(shapes, types))]
    momenta = [torch.zeros(s, device=DEV) for s in shapes]
    copy_of = lambda ts: [t.clone() for t in ts]
    exact, fast, graphed = copy_of(params), copy_of(params), copy_of(params)
    muon_step_(exact, grads, copy_of(momenta), lr=0.02)
    muon_step_(fast, grads, copy_of(momenta), lr=0.02, fast_bf16=True)
    for i, (p, e, f, g) in enumerate(zip(params, exact, fast, grads)):
        big = types[i] == torch.bfloat16 and min(shapes[i]) >= 256
        assert torch.equal(e, f) != big
        want, _ = reference(p, g, 0 * g.double(), 0.02, 0.95, True, 0.1)
        hold(i, f, want, 2.0 ** -9 if big else 2.0 ** -18)
    weights = [torch.nn.Parameter(p.clone()) for p in params]
    opt = Muon([{"params": weights[:3], "fast_bf16": True}, {"params": weights[3:]}], lr=0.02)
    for w, g in zip(weights, grads):
        w.grad = g
    opt.step()
    for i, w in enumerate(weights):
        assert torch.equal(w.detach(), fast[i] if i < 3 else exact[i])
    kept, graph = copy_of(momenta), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon_step_(graphed, grads, kept, lr=0.02, fast_bf16=True)
    for _ in range(3):
        for a, b, m in zip(graphed, params, kept):
            a.copy_(b), m.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, f) for a, f in zip(graphed, fast))


def test_gradients_in_the_momenta_are_refused():
    """They are read again after the momenta are written. (A parameter may be its own gradient.)"""
    p, g = make((40, 30), torch.float32), make((40, 30), torch.float32, seed=1)
    with pytest.raises(ValueError, match="shares memory"):
        muon_step_([p], [g], [g])
    wide = torch.cat([g, g])
    with pytest.raises(ValueError, match="shares memory"):
        muon_step_([p], [wide[:40]], [wide[39:79]])
    q = make((40, 30), torch.float32, seed=2)
    with pytest.raises(ValueError, match="shares memory"):
        muon_step_([p, q], [q, g], [torch.zeros_like(p), torch.zeros_like(p)])
    want, _ = reference(p, p.clone(), torch.zeros_like(p), 0.02, 0.95, True, 0.1)
    muon_step_([p], [p], [torch.zeros_like(p)], lr=0.02)
    hold("p", p, want, REL[torch.float32])
    muon_step_([p, q], [g, g], [torch.zeros_like(p), torch.zeros_like(p)])  # read twice, written nowhere


def test_calls_from_several_threads():
    """Calls at once, on streams of their own."""
    import threading

    x = [make((6, 900, 1030), t) for t in TYPES] + [make((3, 70, 90), torch.float32)]
    want = [orthogonalize(v) for v in x]
    torch.cuda.synchronize()
    got = [None] * len(x)

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(3):
                got[i] = orthogonalize(x[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(x))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for u, v in zip(got, want):
        assert torch.equal(u, v)
