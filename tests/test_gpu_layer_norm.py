"""layer_norm (csrc/layer_norm.hip) against its formula in 64 bits: rows of one element to the widest, odd
widths, more rows than workgroups, with and without weight and bias, strides, rows of one value, NaN and
infinities, other streams and graphs.

Tolerances. In fp32 a mean of d terms, summed by lanes and then across them, is off by 2^-20 of the mean
size, an inverse root by 2^-21, an element less its mean by 2^-20 of the two's sizes; h by 2^-19 of
(|x| + |mean|) rstd, and y and the gradients, sums of products of these, by 2^-17 of the same expressions
with every term by its absolute value (`mag`). Half a step of the type comes on top.
"""
import pytest
import torch

from mambaqc_amd.kernels import layer_norm
from mambaqc_amd.layers import LayerNorm

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
REL, EPS = 2.0 ** -17, 1e-5


def formula(x, w, b, dy=None):
    """name -> (value, magnitude) in 64 bits."""
    x, w, b, dy = (None if v is None else v.detach().double() for v in (x, w, b, dy))
    mean = lambda v: v.mean(-1, keepdim=True)
    w1 = torch.ones_like(x[..., :1]) if w is None else w
    mu = mean(x)
    rstd = (mean((x - mu) ** 2) + EPS).rsqrt()
    h, hm = (x - mu) * rstd, (x.abs() + mean(x.abs())) * rstd
    got = {"y": (h * w1 + (0 if b is None else b), hm * w1.abs() + (0 if b is None else b.abs()))}
    if dy is None:
        return got
    u, um = dy * w1, dy.abs() * w1.abs()
    rows = lambda t: t.reshape(-1, t.shape[-1]).sum(0)
    got |= {"x": (rstd * (u - mean(u) - h * mean(u * h)), rstd * (um + mean(um) + hm * mean(um * hm))),
            "weight": (rows(dy * h), rows(dy.abs() * hm)), "bias": (rows(dy), rows(dy.abs()))}
    return got


def hold(what, got, ref):
    want, mag = ref
    off = (got.double() - want).abs()
    assert got.shape == want.shape, what
    small = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps  # a subnormal's step
    bad = ~(off <= torch.finfo(got.dtype).eps / 2 * want.abs() + REL * mag + small)
    assert not bad.any(), (what, int(bad.sum()), off[bad][:4], want[bad][:4], mag[bad][:4])


def make(shape, dtype, seed=0, weight=True, bias=True):
    gen = torch.Generator(DEV).manual_seed(seed + sum(shape))
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    d = shape[-1]
    x = (2 * r(*shape) + r(*shape[:-1], 1)).to(dtype)
    return x, 1 + 0.3 * r(d) if weight else None, r(d) if bias else None, r(*shape).to(dtype)


def check(x, w, b, dy):
    ref = formula(x, w, b, dy)
    with torch.no_grad():
        y0 = layer_norm(x, w, b, eps=EPS)
    assert y0.dtype == x.dtype
    hold("y", y0, ref["y"])
    leaves = {n: v.detach().requires_grad_() for n, v in (("x", x), ("weight", w), ("bias", b))
              if v is not None}
    y = layer_norm(leaves["x"], leaves.get("weight"), leaves.get("bias"), eps=EPS)
    assert torch.equal(y, y0)
    for (name, leaf), got in zip(leaves.items(), torch.autograd.grad(y, list(leaves.values()), dy)):
        assert got.dtype == leaf.dtype
        hold(name, got, ref[name])


# Around the teams' widths, and more rows than one pass of the workgroups takes.
SHAPES = [(1, 1), (3, 2), (7, 5), (5000, 3), (33, 64), (40, 65), (9, 128), (70, 129), (65, 256), (30, 257),
          (17, 515), (2100, 768), (12, 1000), (3, 1024), (5, 1025), (300, 2048), (7, 4099), (2, 8191),
          (600, 8192), (2, 3, 5, 96)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_values_and_gradients(dtype, shape):
    check(*make(shape, dtype))


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("shape", [(50, 48), (90, 700), (20, 3000)])
def test_without_weight_or_bias(weight, bias, shape):
    check(*make(shape, torch.float32, weight=weight, bias=bias))


@pytest.mark.parametrize("dtype", TYPES)
def test_views_are_read_in_place(dtype):
    wide, w, b, _ = make((4, 30, 200), dtype)
    w, b = w[:96], b[:96]
    for part in (wide[..., :96], wide[..., 103:199], wide[1, :, 5:101], wide[:, 3:4, 7:103],
                 wide.transpose(0, 1)[..., :96], wide[:1, :, :96].expand(3, -1, -1),
                 wide.transpose(1, 2)[..., :96, :].transpose(1, 2)[..., :96]):
        dy = torch.randn(part.shape, device=DEV).to(dtype)
        check(part, w, b, dy)
    dy = torch.randn(4, 96, 30, device=DEV).to(dtype).transpose(1, 2)
    check(wide[..., :96], w, b, dy)


def test_rows_of_one_value_and_far_means():
    x, w, b, dy = make((20, 300), torch.float32)
    x[3] = 0.0
    x[4] = 7.0
    x[5] += 1000.0
    x[6] *= 1e-12
    x[7] *= 1e15
    check(x, w, b, dy)


def test_nan_and_infinities_stay_in_their_rows():
    for d in (64, 768, 3000):
        x, w, b, dy = make((9, d), torch.float32)
        x[2, 1], x[5, 0], dy[7, d - 1] = float("nan"), float("inf"), float("nan")
        x.requires_grad_()
        y = layer_norm(x, w, b)
        dx, = torch.autograd.grad(y, x, dy)
        fine = [0, 1, 3, 4, 6, 8]
        assert y[fine].isfinite().all() and dx[fine].isfinite().all()
        assert y[2].isnan().all() and y[5].isnan().any() and y[7].isfinite().all() and dx[7].isnan().all()


def test_gradients_against_differences():
    x, w, b, dy = make((11, 70), torch.float32)
    leaves = [v.requires_grad_() for v in (x, w, b)]
    grads = torch.autograd.grad(layer_norm(*leaves), leaves, dy)
    step = 2.0 ** -6
    with torch.no_grad():
        for i, (v, grad) in enumerate(zip(leaves, grads)):
            way = torch.randn(v.shape, generator=torch.Generator(DEV).manual_seed(i), device=DEV)
            ends = [(layer_norm(*[u + sign * step * way if u is v else u for u in leaves]).double() * dy).sum()
                    for sign in (1, -1)]
            slope, along = (ends[0] - ends[1]) / (2 * step), (grad.double() * way).sum()
            # Third derivatives times step^2 / 6, and the values' rounding over 2 step.
            size = (grad.double() * way).norm() + 2.0 ** -13 * dy.double().norm()
            assert (slope - along).abs() <= 2e-2 * size, (i, slope, along)


def test_empty_and_mixed_types():
    w = torch.ones(8, device=DEV, requires_grad=True)
    x = torch.empty(0, 8, device=DEV, requires_grad=True)
    y = layer_norm(x, w, w)
    assert y.shape == (0, 8)
    got = torch.autograd.grad(y, [x, w], torch.ones_like(y))
    assert got[0].shape == (0, 8) and (got[1] == 0).all()
    assert layer_norm(torch.empty(3, 0, device=DEV)).shape == (3, 0)
    x, w, b, dy = make((30, 100), torch.float16)
    check(x, w.bfloat16(), b.half(), dy)


def test_module():
    x, _, _, dy = make((4, 20, 96), torch.bfloat16)
    ours, theirs = LayerNorm(96).to(DEV), torch.nn.LayerNorm(96).to(DEV)
    torch.nn.init.normal_(theirs.weight)
    torch.nn.init.normal_(theirs.bias)
    ours.load_state_dict(theirs.state_dict())
    hold("y", ours(x).detach(), formula(x, theirs.weight, theirs.bias)["y"])
    ours(x).backward(dy)
    ref = formula(x, theirs.weight, theirs.bias, dy)
    hold("weight", ours.weight.grad, ref["weight"])
    hold("bias", ours.bias.grad, ref["bias"])
    plain = LayerNorm(96, elementwise_affine=False).to(DEV)
    hold("y", plain(x), formula(x, None, None)["y"])
    with pytest.raises(ValueError, match="expected"):
        ours(x[..., :95])


def test_repeats_streams_and_graphs():
    x, w, b, dy = make((3000, 515), torch.bfloat16)
    leaves = [v.requires_grad_() for v in (x, w, b)]
    once = lambda: [y := layer_norm(*leaves), *torch.autograd.grad(y, leaves, dy)]
    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = once()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(u, v) for u, v in zip(first, other))
    del first, other
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [v.detach() for v in once()]
    for rep in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=torch.Generator(DEV).manual_seed(rep), device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in outs]
        assert all(torch.equal(u, v) for u, v in zip(got, once())), rep


def test_compiles():
    x, w, b, dy = make((3, 20, 48), torch.float32)
    leaves = [v.requires_grad_() for v in (x, w, b)]
    fn = lambda *v: layer_norm(*v) * 2.0
    want = fn(*leaves)
    got = torch.compile(fn, backend="aot_eager", fullgraph=True)(*leaves)
    assert torch.equal(got, want)
    for a, c in zip(torch.autograd.grad(got, leaves, dy), torch.autograd.grad(want, leaves, dy)):
        assert torch.equal(a, c)
    y = torch.compile(lambda v: layer_norm(v), backend="aot_eager", fullgraph=True)(x)
    assert torch.equal(y, layer_norm(x))


def test_second_and_forward_gradients_are_refused():
    x, w, b, dy = make((3, 20), torch.float32)
    x.requires_grad_()
    dx, = torch.autograd.grad(layer_norm(x, w, b), x, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="gradient of the gradient"):
        dx.sum().backward()
    ad = torch.autograd.forward_ad
    with ad.dual_level():
        with pytest.raises(RuntimeError):
            layer_norm(ad.make_dual(x.detach(), torch.ones_like(x)), w, b)


@pytest.mark.parametrize("hooks", [torch.autograd.graph.save_on_cpu, lambda: torch.autograd.graph.saved_tensors_hooks(
    lambda t: t.mT.contiguous().mT if t.dim() > 1 else t.clone(), lambda t: t)])
def test_saved_tensors_come_back_laid_out_anew(hooks):
    wide, w, b, dy = make((3, 40, 96), torch.float32)
    x, w, b = wide[..., 10:50].detach().requires_grad_(), w[:40].detach().requires_grad_(), b[:40].clone()
    want = torch.autograd.grad(layer_norm(x, w, b), [x, w], dy[..., :40])
    with hooks():
        y = layer_norm(x, w, b)
    for a, c in zip(torch.autograd.grad(y, [x, w], dy[..., :40]), want):
        assert torch.equal(a, c)


def test_offsets_past_32_bits():
    """Rows more than 2^32 bytes into their tensors: the last ones alone."""
    x = torch.empty(2_200_000, 1024, device=DEV, dtype=torch.bfloat16).normal_()
    w = torch.linspace(-1, 1, 1024, device=DEV)
    x.requires_grad_()
    y = layer_norm(x, w)
    dx, = torch.autograd.grad(y, x, x.detach())
    tail = x[-300:].detach().clone()
    ref = formula(tail, w, None, tail)
    hold("y", y[-300:].detach(), ref["y"])
    hold("x", dx[-300:], ref["x"])


def test_registered_backward_checks_what_it_reads():
    x, w, b, dy = make((5, 24), torch.float32)
    op = torch.ops.mambaqc.layer_norm_backward
    stats = torch.ops.mambaqc.layer_norm(x, w, b)[1]
    op(x, w, b, stats, dy)
    for bad in ((stats[:4], dy), (stats, dy[:4])):
        with pytest.raises(ValueError, match="must be"):
            op(x, w, b, *bad)
