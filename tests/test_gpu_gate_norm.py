"""gate_norm_residual (csrc/gate_norm.hip) against its formula in 64 bits: rows of one element to the
widest, odd widths, more rows than workgroups, with and without gate and post norm, strides, rows of
zeros, NaN and infinities, each output alone, other streams and graphs.

Tolerances. In fp32 the gate is off by 2^-21 of itself (the exponential's rounded argument for |z| up to
8), a norm by 2^-21 (a sum of squares), a product of those with a weight by 2^-19 of its size, and a
sum of such products by 2^-19 of the sum of their sizes (`mag`: every term by its absolute value). The
norm of out carries out's error: 2^-19 of mag's norm over out's, at most 4 for these inputs. Gradients
multiply two of these: 2^-16 of their mag covers all, and half a step of the type comes on top.
"""
import pytest
import torch

from mambaqc_amd.kernels import gate_norm_residual

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
REL = 2.0 ** -16
EPS = 1e-6


def formula(x, y, z, post, scale, pre, dout=None, dn=None):
    """name -> (value, magnitude) in 64 bits."""
    x, y, z, post, scale, pre, dout, dn = (None if v is None else v.detach().double()
                                           for v in (x, y, z, post, scale, pre, dout, dn))
    mean = lambda v: v.mean(-1, keepdim=True)
    gate = torch.sigmoid(z) if z is not None else torch.ones_like(y)
    v = gate * y
    rho = (mean(v * v) + EPS).rsqrt() if post is not None else torch.ones_like(mean(v))
    p = post if post is not None else torch.ones_like(scale)
    r = v * rho * p
    o, om = x + scale * r, x.abs() + (scale * r).abs()
    tau = (mean(o * o) + EPS).rsqrt()
    got = {"out": (o, om), "n": (o * tau * pre, om * tau * pre.abs())}
    if dn is None:
        return got
    u, w = dn * pre, scale * p
    O = dout + tau * u - o * tau ** 3 * mean(u * o)
    Om = dout.abs() + tau * u.abs() + om * tau ** 3 * mean(u.abs() * om)
    dv, dvm = rho * w * O, rho * w.abs() * Om
    if post is not None:
        dv = dv - v * rho ** 3 * mean(w * O * v)
        dvm = dvm + v.abs() * rho ** 3 * mean(w.abs() * Om * v.abs())
    rows = lambda t: t.reshape(-1, t.shape[-1]).sum(0)
    got |= {"x": (O, Om), "y": (dv * gate, dvm * gate),
            "scale": (rows(O * r), rows(Om * r.abs())),
            "pre": (rows(dn * o * tau), rows(dn.abs() * om * tau))}
    if z is not None:
        got["z"] = (dv * v * torch.sigmoid(-z), dvm * v.abs() * torch.sigmoid(-z))
    if post is not None:
        got["post"] = (rows(scale * O * v * rho), rows(scale.abs() * Om * v.abs() * rho))
    return got


def hold(what, got, ref):
    want, mag = ref
    off = (got.double() - want).abs()
    assert got.shape == want.shape, what
    small = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps  # a subnormal's step
    bad = ~(off <= torch.finfo(got.dtype).eps / 2 * want.abs() + REL * mag + small)
    assert not bad.any(), (what, int(bad.sum()), off[bad][:4], want[bad][:4], mag[bad][:4])


def make(shape, dtype, gate=True, post=True, seed=0):
    d = shape[-1]
    gen = torch.Generator(device=DEV).manual_seed(seed + sum(shape))
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    return {"x": r(*shape).to(dtype), "y": r(*shape).to(dtype),
            "z": r(*shape[:-1], 2 * d)[..., d:].to(dtype) if gate else None,
            "post": 1 + 0.2 * r(d) if post else None, "scale": 0.3 + 0.1 * r(d),
            "pre": 1 + 0.2 * r(d)}, r(*shape).to(dtype), r(*shape).to(dtype)


def call(v, eps=EPS):
    return gate_norm_residual(v["x"], v["y"], v["z"], post_weight=v["post"], scale=v["scale"],
                              pre_weight=v["pre"], eps=eps)


def check(v, dout, dn):
    ref = formula(*v.values(), dout, dn)
    with torch.no_grad():
        first = call(v)
    for name, got in zip(("out", "n"), first):
        hold(name, got, ref[name])
    leaves = {k: t.detach().requires_grad_() for k, t in v.items() if t is not None}
    outs = call({**v, **leaves})
    for a, b in zip(first, outs):
        assert torch.equal(a, b)
    for name, got in zip(leaves, torch.autograd.grad(outs, list(leaves.values()), [dout, dn])):
        assert got.dtype == leaves[name].dtype
        hold(name, got, ref[name])


# Rows x width: single elements, around a lane's 4, a wave's 256 to 1024, a workgroup's, the widest;
# more rows than the backward has workgroups.
SIZES = [(1, 1), (3, 2), (5, 3), (2, 4), (9, 17), (7, 255), (9, 256), (6, 257), (40, 515), (5, 768),
         (33, 1023), (9, 1024), (3, 1025), (2, 2047), (3, 4096), (3, 4097), (2, 8191), (2, 8192),
         (2101, 65), (1500, 300), (600, 1500)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,d", SIZES)
@pytest.mark.parametrize("gate,post", [(True, True), (False, False)])
def test_values_and_gradients(dtype, rows, d, gate, post):
    check(*make((rows, d), dtype, gate, post))


@pytest.mark.parametrize("gate,post", [(True, False), (False, True)])
@pytest.mark.parametrize("shape", [(2, 3, 100), (1, 700), (13,)])
def test_parts_and_shapes(shape, gate, post):
    check(*make(shape, torch.bfloat16, gate, post))


@pytest.mark.parametrize("which", [0, 1])
def test_one_output_alone(which):
    v, dout, dn = make((20, 130), torch.float32)
    zero = torch.zeros_like(dout)
    ref = formula(*v.values(), zero if which else dout, dn if which else zero)
    leaves = {k: t.detach().requires_grad_() for k, t in v.items()}
    got = torch.autograd.grad(call(leaves)[which], list(leaves.values()), (dout, dn)[which],
                              allow_unused=True)
    for name, g in zip(leaves, got):
        hold(name, g, ref[name])


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_zeros_are_finite(dtype):
    """Norms of nothing but eps; rows beside them are not touched."""
    v, dout, dn = make((6, 70), dtype)
    v["x"][1], v["y"][1], v["y"][2], v["x"][4] = 0, 0, 0, 0
    # Two norms of 1 / sqrt(eps) multiply such a row's gradients by 1e6: small ones keep within fp16.
    check(v, dout / 256, dn / 256)


@pytest.mark.parametrize("d", [90, 300, 1100])
def test_nan_and_inf_stay_in_their_row(d):
    v, dout, dn = make((7, d), torch.float32)
    want = formula(*v.values(), dout, dn)
    v["x"][2, 5], v["y"][3, 7], v["z"][4, d - 1] = float("nan"), float("inf"), float("nan")
    leaves = {k: v[k].detach().requires_grad_() for k in ("x", "y", "z")}
    out, n = call({**v, **leaves})
    ok = [0, 1, 5, 6]
    for got, name in zip((out, n, *torch.autograd.grad([out, n], list(leaves.values()), [dout, dn])),
                         ("out", "n", "x", "y", "z")):
        hold(name, got[ok], tuple(t[ok] for t in want[name]))
    assert n[[2, 3, 4]].isnan().any(1).all()


def test_gates_at_the_ends_of_their_type():
    v, dout, dn = make((4, 64), torch.float32)
    v["z"] = torch.tensor([-1e30, -100.0, 100.0, 1e30], device=DEV)[:, None].repeat(1, 64)
    leaves = {k: t.detach().requires_grad_() for k, t in v.items()}
    out, n = call(leaves)
    ref = formula(*v.values(), dout, dn)
    hold("out", out[2:], tuple(t[2:] for t in ref["out"]))
    assert torch.equal(out[0], v["x"][0])
    for g in torch.autograd.grad([out, n], list(leaves.values()), [dout, dn]):
        assert g.isfinite().all()


@pytest.mark.parametrize("d", [64, 37])
def test_strides_and_broadcasts(d):
    v, dout, dn = make((2, 30, d), torch.bfloat16)
    want = call({k: None if t is None else t.clone() for k, t in v.items()})
    turned = {k: v[k].transpose(0, 1).contiguous().transpose(0, 1) for k in ("x", "y", "z")}
    for a, b in zip(call({**v, **turned}), want):
        assert torch.equal(a, b)
    # A row that all rows share: its gradient is the sum.
    row = v["x"][:1, :1].float().requires_grad_()
    w = {**v, "x": row.expand(2, 30, -1)}
    out, n = call(w)
    assert out.dtype == torch.float32
    ref = formula(*w.values(), dout.float(), dn.float())
    hold("x", torch.autograd.grad([out, n], row, [dout.float(), dn.float()])[0],
         tuple(t.sum((0, 1), keepdim=True) for t in ref["x"]))


def test_gradients_against_differences():
    v, dout, dn = make((3, 40), torch.float32)
    leaves = {k: t.detach().requires_grad_() for k, t in v.items()}
    grads = torch.autograd.grad(call(leaves), list(leaves.values()), [dout, dn])
    step = 2.0 ** -8
    with torch.no_grad():
        for i, (k, g) in enumerate(zip(leaves, grads)):
            way = torch.randn(g.shape, generator=torch.Generator(DEV).manual_seed(i), device=DEV)
            ends = []
            for sign in (1, -1):
                out, n = call({**v, k: v[k] + sign * step * way})
                ends.append((out.double() * dout + n.double() * dn).sum())
            slope, along = (ends[0] - ends[1]) / (2 * step), (g.double() * way).sum()
            # Third derivatives times step^2 / 6, and the values' 2^-19 over 2 step.
            size = (g.double() * way).norm() + 2.0 ** -11 * (dout.norm() + dn.norm())
            assert (slope - along).abs() <= 1e-2 * size, (k, slope, along)


def test_mixed_types_and_16_bit_weights():
    v, dout, dn = make((5, 50), torch.float16)
    v["y"] = v["y"].float()
    for k in ("post", "scale", "pre"):
        v[k] = v[k].bfloat16()
    check(v, dout.float(), dn.float())


def test_no_rows():
    v, _, _ = make((0, 8), torch.bfloat16)
    leaves = {k: t.detach().requires_grad_() for k, t in v.items()}
    out, n = call(leaves)
    assert out.shape == n.shape == (0, 8)
    for k, g in zip(leaves, torch.autograd.grad([out, n], list(leaves.values()), [out, n])):
        assert g.shape == leaves[k].shape and (g == 0).all()


def test_too_wide_is_refused():
    x, w = torch.zeros(2, 8193, device=DEV), torch.zeros(8193, device=DEV)
    with pytest.raises(RuntimeError, match="mqc_gate_norm_fwd"):
        gate_norm_residual(x, x, scale=w, pre_weight=w)


def test_other_streams_repeats_and_graphs():
    v, dout, dn = make((1300, 200), torch.bfloat16)
    leaves = {k: t.detach().clone().requires_grad_() for k, t in v.items()}

    def once():
        outs = call(leaves)
        return [*outs, *torch.autograd.grad(outs, list(leaves.values()), [dout, dn])]

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, other):
        assert torch.equal(a, b)
    del first, other
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [t.detach() for t in once()]
    for rep in range(4):
        with torch.no_grad():
            leaves["y"].copy_(torch.randn(1300, 200, generator=torch.Generator(DEV).manual_seed(rep),
                                          device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        for a, b in zip(got, once()):
            assert torch.equal(a, b), rep


@pytest.mark.parametrize("gate,post", [(True, True), (False, False)])
def test_registered_operators(gate, post):
    v, dout, dn = make((2, 9, 40), torch.float32, gate, post)
    leaves = {k: None if t is None else t.detach().requires_grad_() for k, t in v.items()}
    out, n, _ = torch.ops.mambaqc.gate_norm_residual(*leaves.values(), EPS)
    want = call(leaves)
    assert torch.equal(out, want[0]) and torch.equal(n, want[1])
    some = [t for t in leaves.values() if t is not None]
    for a, b in zip(torch.autograd.grad([out, n], some, [dout, dn]),
                    torch.autograd.grad(want, some, [dout, dn])):
        assert torch.equal(a, b)


def test_more_than_the_caches_hold():
    """Outputs stored past the caches (over 256 MiB in all)."""
    v, _, _ = make((14000, 1026), torch.float32)
    ref = formula(*v.values())
    with torch.no_grad():
        for name, got in zip(("out", "n"), call(v)):
            hold(name, got, ref[name])


def test_second_gradients_are_refused():
    v, dout, _ = make((4, 30), torch.float32)
    x = v["x"].requires_grad_()
    dx, = torch.autograd.grad(call(v)[0], x, dout, create_graph=True)
    with pytest.raises(RuntimeError, match="gradient of the gradient"):
        dx.sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows,d", [(1, 16), (17, 63), (33, 64), (70, 66), (9, 127), (31, 128), (5, 129),
                                    (20000, 30), (9000, 110)])
def test_narrow_rows(dtype, rows, d):
    """Teams of 16, 32 and 64 lanes, their last ones without a row."""
    check(*make((rows, d), dtype))


def test_offsets_past_32_bits():
    """The last rows of tensors of more than 2^32 bytes equal those rows alone, bit for bit."""
    rows, d = 2_200_000, 1000
    r = lambda *s: torch.empty(*s, device=DEV, dtype=torch.bfloat16).normal_()
    v = {"x": r(rows, d), "y": r(rows, d), "z": r(rows, d + 40)[:, 40:], "post": torch.ones(d, device=DEV),
         "scale": torch.full((d,), 0.5, device=DEV), "pre": torch.ones(d, device=DEV)}
    dout, dn = r(rows, d), r(rows, d)
    end = {k: t[-50:] if t.dim() == 2 else t for k, t in v.items()}
    results = []
    for w, gs in ((v, [dout, dn]), (end, [dout[-50:], dn[-50:]])):
        leaves = {k: t.detach().requires_grad_(k in "xyz") for k, t in w.items()}
        outs = call(leaves)
        results.append([*outs, *torch.autograd.grad(outs, [leaves[k] for k in "xyz"], gs)])
    for a, b in zip(*results):
        assert torch.equal(a[-50:], b)


def test_compiles():
    """Traced through the registered operators, with the same results."""
    v, dout, dn = make((30, 70), torch.float32)
    leaves = {k: t.detach().requires_grad_() for k, t in v.items()}
    fn = lambda *t: call(dict(zip(v, t)))
    want = fn(*leaves.values())
    got = torch.compile(fn, backend="aot_eager", fullgraph=True)(*leaves.values())
    some = list(leaves.values())
    for a, b in zip([*got, *torch.autograd.grad(got, some, [dout, dn])],
                    [*want, *torch.autograd.grad(want, some, [dout, dn])]):
        assert torch.equal(a, b)


def copies(order):
    """Hooks on saved tensors that give back dense copies, or ones whose axes lie in another order."""
    def pack(t):
        kept = torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)
        return kept if order == "dense" or t.dim() < 2 else kept.transpose(0, 1).contiguous().transpose(0, 1)
    return torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t)


@pytest.mark.parametrize("hooks", [lambda: copies("dense"), lambda: copies("turned"),
                                   torch.autograd.graph.save_on_cpu])
@pytest.mark.parametrize("shape", [(1, 40), (50, 40), (30, 515), (2, 3, 300)])
def test_saved_tensors_come_back_laid_out_anew(hooks, shape):
    """The backward reads what hooks on saved tensors give back, not the forward's rows."""
    v, dout, dn = make(shape, torch.float32)
    wide = torch.randn(*shape[:-1], 3 * shape[-1], device=DEV)

    def grads():
        leaves = {k: t.detach().requires_grad_() for k, t in v.items() if k != "z"}
        leaf = wide.detach().requires_grad_()
        outs = call({**leaves, "z": leaf[..., shape[-1]:2 * shape[-1]]})
        return torch.autograd.grad(outs, [leaf, *leaves.values()], [dout, dn])

    want = grads()
    with hooks():
        got = grads()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_saved_tensors_of_other_shapes_are_refused():
    v, dout, dn = make((30, 40), torch.float32)
    v["x"].requires_grad_()
    for shape in [(30, 40), (40,), (30, 2)]:
        with torch.autograd.graph.saved_tensors_hooks(
                lambda t: t, lambda t: t[:1] if tuple(t.shape) == shape else t):
            out, n = call(v)
        with pytest.raises(ValueError, match="must be|other shapes"):
            (out * dout + n * dn).sum().backward()


def test_registered_backward_checks_what_it_reads():
    v, dout, dn = make((30, 40), torch.float32)
    ops = (v["x"], v["y"], v["z"], v["post"], v["scale"], v["pre"])
    stats = torch.ops.mambaqc.gate_norm_residual(*ops)[2]
    op = torch.ops.mambaqc.gate_norm_residual_backward
    op(*ops, stats, dout, dn)
    for bad in ((stats[:29], dout, dn), (stats, dout[:29], dn), (stats, dout, dn[:, :39])):
        with pytest.raises(ValueError, match="must be"):
            op(*ops, *bad)
    with pytest.raises(RuntimeError, match="ROCm device"):
        op(*ops, stats.cpu(), dout, dn)


def test_forward_mode_is_refused():
    v, dout, _ = make((4, 40), torch.float32)
    x = v["x"].requires_grad_()
    out = call(v)[0]
    ad = torch.autograd.forward_ad
    with ad.dual_level():
        for grad in (False, True):
            dual = ad.make_dual(x.detach().requires_grad_(grad), torch.ones_like(x))
            with pytest.raises(RuntimeError):
                call({**v, "x": dual})
        with pytest.raises(RuntimeError):  # a gradient with a tangent
            torch.autograd.grad(out, x, ad.make_dual(dout, torch.ones_like(dout)))
    assert call(v)[1].isfinite().all()


@pytest.mark.parametrize("d", [40, 300, 1500, 5000])
@pytest.mark.parametrize("gate", [True, False])
def test_rows_near_zero_under_a_small_eps(d, gate, monkeypatch):
    """Inverse norms up to 1e15, whose cubes fp32 does not hold: rows of zeros (padding) and tiny ones."""
    monkeypatch.setitem(globals(), "EPS", 1e-30)
    v, dout, dn = make((6, d), torch.float32, gate)
    size = torch.tensor([0.0, 1e-16, 1e-14, 1.0, 0.0, 1e-10], device=DEV)[:, None]
    v["x"], v["y"] = v["x"] * size, v["y"] * size
    ref = formula(*v.values(), dout, dn)
    leaves = {k: t.detach().requires_grad_() for k, t in v.items() if t is not None}
    outs = call({**v, **leaves}, eps=EPS)
    for name, got in zip(("out", "n"), outs):
        hold(name, got.detach(), ref[name])
    for name, got in zip(leaves, torch.autograd.grad(outs, list(leaves.values()), [dout, dn])):
        assert got.isfinite().all(), name
        hold(name, got, ref[name])
