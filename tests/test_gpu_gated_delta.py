"""The gated delta rule (csrc/gated_delta.hpp) against the recurrence walked in 64 bits: values, states and
gradients at sizes around its chunks and tiles, shared key heads, resets, strides, decays from none to
all, the single-token step, NaN behind a reset, other streams and graphs.

Tolerances. With keys of length one and beta in [0, 1] a token's map of the state does not lengthen it, so
errors add up and do not grow. An output is a sum of n = k_dim + 64 + 64 products of fp32 values (a
state's columns, a chunk's tokens, the triangular system), each off by a few 2^-24 of its size, and what
they are off by adds up as its square does: 2^-22 sqrt(n) = 2^-18 of the products' size, once for each of
the chunks that a value has come through, at most 16 here, again as squares: 2^-16. Gradients are products
of two such results: 2^-15. Sizes are the tensor's: an element is held to REL times the larger of itself
and four times the root mean square (that of single elements at 1 x 1 sizes), plus half a step of its type.
"""
import pytest
import torch

from mambaqc_amd import _native as nat
from mambaqc_amd.kernels import gated_delta, gated_delta_step_

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
REL, GRAD = 2.0 ** -16, 2.0 ** -15
NAMES = ("q", "k", "v", "g", "beta", "h0")


def walk(q, k, v, g, beta, h0, reset, scale=None):
    """(o, last state) from 64-bit operands, token by token, differentiable."""
    group = v.shape[2] // q.shape[2]
    scale = q.shape[3] ** -0.5 if scale is None else scale
    q, k = (x.repeat_interleave(group, 2) for x in (q, k))
    b, t, h, dv = v.shape
    S = v.new_zeros(b, h, q.shape[3], dv) if h0 is None else h0
    out = []
    for i in range(t):
        p = S * g[:, i].exp()[..., None, None]
        if reset is not None:
            p = torch.where(reset[:, i, None, None, None], 0.0, p)
        r = v[:, i] - (p * k[:, i, :, :, None]).sum(2)
        S = p + k[:, i, :, :, None] * (beta[:, i, :, None] * r)[:, :, None]
        out.append(scale * (S * q[:, i, :, :, None]).sum(2))
    return (torch.stack(out, 1) if out else v), S


def exact(ops, reset, do, dh, scale=None):
    """name -> value in 64 bits, gradients by differentiating the walk."""
    leaves = [None if x is None else x.detach().double().requires_grad_() for x in ops]
    o, h = walk(*leaves, reset, scale)
    got = {"o": o.detach(), "h": h.detach()}
    some = [x for x in leaves if x is not None]
    grads = torch.autograd.grad([o, h], some, [do.double(), dh.double()])
    return got | dict(zip([n for n, x in zip(NAMES, leaves) if x is not None], grads))


def hold(what, got, want, rel):
    assert got.shape == want.shape, what
    half = torch.finfo(got.dtype).eps / 2
    off, rms = (got.double() - want).abs(), want.square().mean().sqrt()
    bad = ~(off <= half * want.abs() + rel * torch.maximum(want.abs(), 4 * rms)
            + torch.finfo(got.dtype).smallest_normal)
    assert not bad.any(), (what, int(bad.sum()), off[bad][:4], want[bad][:4], rms)


def make(b, t, hk, hv, dk, dv, dtype, seed=0, h0=True, reset=0.0, rate=0.3):
    gen = torch.Generator(device=DEV).manual_seed(seed + 7 * b + 11 * t + 13 * dk + 17 * dv)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    unit = lambda x: (x / x.norm(dim=-1, keepdim=True)).to(dtype)
    q, k, v = unit(r(b, t, hk, dk)), unit(r(b, t, hk, dk)), r(b, t, hv, dv).to(dtype)
    g = -rate * torch.rand(b, t, hv, generator=gen, device=DEV) ** 3
    beta = torch.sigmoid(r(b, t, hv)).to(dtype)
    cut = torch.rand(b, t, generator=gen, device=DEV) < reset if reset else None
    ops = [q, k, v, g, beta, r(b, hv, dk, dv) if h0 else None]
    return ops, cut, r(b, t, hv, dv).to(dtype), r(b, hv, dk, dv)


def check(ops, cut, do, dh, scale=None):
    ref = exact(ops, cut, do, dh, scale)
    with torch.no_grad():
        o0, h0 = gated_delta(*ops[:5], h0=ops[5], reset=cut, scale=scale, return_state=True)
    hold("o", o0, ref["o"], REL)
    hold("h", h0, ref["h"], REL)
    leaves = [None if x is None else x.detach().requires_grad_() for x in ops]
    o, h = gated_delta(*leaves[:5], h0=leaves[5], reset=cut, scale=scale, return_state=True)
    assert torch.equal(o, o0) and torch.equal(h, h0)
    some = [x for x in leaves if x is not None]
    names = [n for n, x in zip(NAMES, leaves) if x is not None]
    for name, leaf, got in zip(names, some, torch.autograd.grad([o, h], some, [do, dh])):
        assert got.dtype == leaf.dtype
        hold(name, got, ref[name], GRAD)
    return o0, h0


# Around a chunk of 64 tokens, key widths of 32, 64 and 128 and tiles of 16 and 32 columns; odd sizes.
SIZES = [(1, 1, 1, 1, 1, 1), (2, 2, 1, 1, 16, 16), (1, 63, 2, 2, 33, 17), (2, 64, 1, 3, 64, 64),
         (1, 65, 2, 4, 60, 100), (3, 130, 1, 1, 128, 130), (1, 200, 3, 3, 100, 20), (1, 1000, 1, 2, 31, 40)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("state,reset", [(False, 0.0), (True, 0.04)])
def test_values_and_gradients(dtype, size, state, reset):
    check(*make(*size, dtype, h0=state, reset=reset))


@pytest.mark.parametrize("at", [[0], [63], [64], [65], [1, 2, 3], [10, 64, 100], list(range(130))])
def test_resets(at):
    ops, _, do, dh = make(2, 130, 1, 2, 20, 24, torch.float32)
    cut = torch.zeros(2, 130, dtype=torch.bool, device=DEV)
    cut[0, at] = True
    o, h = check(ops, cut, do, dh)
    start = at[-1]  # the last document alone
    part = [x[:1, start:] for x in ops[:5]]
    o1, h1 = gated_delta(*part, return_state=True)
    hold("o", o[:1, start:], o1.double(), REL)
    hold("h", h[:1], h1.double(), REL)


@pytest.mark.parametrize("dtype", TYPES)
def test_decays_and_rates_at_their_ends(dtype):
    """No decay, decays that underflow, total ones, and beta 0, 1 and 2 (a reflection)."""
    ops, _, do, dh = make(1, 150, 2, 2, 24, 33, dtype)
    g, beta = ops[3], ops[4]
    g[:, :, 0] = 0.0
    g[:, 5::17, 1] = -200.0
    g[:, 9::31, 1] = -1e6
    g[:, 70, 1] = -float("inf")
    beta[:, 3::5] = 0.0
    beta[:, 4::5] = 1.0
    beta[:, 7::20] = 2.0
    ref = [x.clone() for x in ops]
    ref[3] = g.clamp_min(-700.0)  # exp of it is 0 to 64 bits too, and its slope a number
    want = exact(ref, None, do, dh)
    leaves = [x.detach().requires_grad_() for x in ops]
    o, h = gated_delta(*leaves[:5], h0=leaves[5], return_state=True)
    hold("o", o.detach(), want["o"], REL)
    hold("h", h.detach(), want["h"], REL)
    for name, got in zip(NAMES, torch.autograd.grad([o, h], leaves, [do, dh])):
        hold(name, got, want[name], GRAD)


def test_long_slow_state_and_scale():
    ops, _, do, dh = make(1, 1024, 1, 1, 128, 32, torch.bfloat16, rate=1e-3)
    check(ops, None, do, dh, scale=1.5)


@pytest.mark.parametrize("which", ["o", "h"])
def test_one_output_alone(which):
    ops, cut, do, dh = make(2, 100, 1, 2, 20, 40, torch.float32, reset=0.02)
    ref = exact(ops, cut, do if which == "o" else 0 * do, dh if which == "h" else 0 * dh)
    leaves = [x.detach().requires_grad_() for x in ops]
    o, h = gated_delta(*leaves[:5], h0=leaves[5], reset=cut, return_state=True)
    got = torch.autograd.grad(o if which == "o" else h, leaves, do if which == "o" else dh)
    for name, v in zip(NAMES, got):
        hold(name, v, ref[name], GRAD)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dk,dv", [(64, 32), (30, 33)])
def test_views_are_read_in_place(dtype, dk, dv):
    """Parts of one projection's output at odd places, heads before tokens, a broadcast batch and key."""
    ops, _, do, dh = make(2, 70, 2, 4, dk, dv, dtype)
    o, h = check(ops, None, do, dh)
    wide = torch.cat([x.flatten(2) for x in ops[:3]] + [do.flatten(2)[..., :3]], -1)
    q = wide[..., :2 * dk].unflatten(-1, (2, dk))
    k = wide[..., 2 * dk:4 * dk].unflatten(-1, (2, dk))
    v = wide[..., 4 * dk:4 * dk + 4 * dv].unflatten(-1, (4, dv))
    assert torch.equal(gated_delta(q, k, v, *ops[3:5], h0=ops[5]), o)
    turned = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in ops[:5]]
    assert torch.equal(gated_delta(*turned, h0=ops[5]), o)
    last = [x.transpose(2, 3).contiguous().transpose(2, 3) for x in ops[:3]]
    assert torch.equal(gated_delta(*last, *ops[3:5], h0=ops[5]), o)
    one = [x[:1].expand(2, *x.shape[1:]) for x in ops]
    assert torch.equal(gated_delta(*one[:5], h0=one[5])[1], o[0])
    # A key for every head: its gradient is the sum over them.
    leaf = ops[1][:, :, :1].detach().requires_grad_()
    spread = gated_delta(ops[0], leaf.expand(2, 70, 2, dk), ops[2], *ops[3:5])
    got, = torch.autograd.grad(spread, leaf, do)
    want = exact([ops[0], ops[1][:, :, :1].expand(2, 70, 2, dk), ops[2], *ops[3:5], None], None, do, 0 * dh)
    hold("k", got, want["k"].sum(2, keepdim=True), GRAD + torch.finfo(dtype).eps)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(1, 1, 1, 1, 1), (3, 2, 4, 60, 101), (16, 2, 2, 128, 128), (2, 1, 3, 17, 300)])
def test_step(dtype, size):
    b, hk, hv, dk, dv = size
    ops, _, _, _ = make(b, 5, hk, hv, dk, dv, dtype)
    want, last = walk(*(x.double() for x in ops), None)
    h = ops[5].clone()
    for i in range(5):
        o = gated_delta_step_(*(x[:, i:i + 1] for x in ops[:5]), h)
        hold("o", o[:, 0], want[:, i], REL)
    hold("h", h, last, REL)
    o, h1 = gated_delta(*ops[:5], h0=ops[5], return_state=True)
    hold("h", h1, last, REL)


def test_state_continues_a_split_sequence():
    ops, cut, _, _ = make(2, 300, 2, 2, 40, 48, torch.float32, reset=0.01)
    o, h = gated_delta(*ops[:5], h0=ops[5], reset=cut, return_state=True)
    state, parts = ops[5], []
    for start, end in ((0, 1), (1, 70), (70, 134), (134, 300)):
        some, state = gated_delta(*(x[:, start:end] for x in ops[:5]), h0=state, reset=cut[:, start:end],
                                  return_state=True)
        parts.append(some)
    hold("o", torch.cat(parts, 1), o.double(), REL)
    hold("h", state, h.double(), REL)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("what", range(6))
@pytest.mark.parametrize("at,first", [(20, 40), (20, 64), (63, 64), (70, 150), (20, 21)])
def test_nan_stays_before_a_reset(bad, what, at, first):
    """A document that is not finite (or the state before it) leaves the next one's outputs and last state
    as they are, and gradients from 64 tokens on."""
    ops, _, do, dh = make(1, 260, 1, 2, 40, 24, torch.float32)
    cut = torch.zeros(1, 260, dtype=torch.bool, device=DEV)
    cut[0, first] = True
    good = gated_delta(*ops[:5], h0=ops[5], reset=cut, return_state=True)
    (ops[5] if what == 5 else ops[what][0, at])[..., 0] = bad
    leaves = [x.requires_grad_() for x in ops]
    o, h = gated_delta(*leaves[:5], h0=leaves[5], reset=cut, return_state=True)
    hold("o", o[:, first:].detach(), good[0][:, first:].double(), REL)
    hold("h", h.detach(), good[1].double(), REL)
    if at >= 64 or what == 5:  # chunks before it
        assert what == 5 or o[:, :64].isfinite().all()
    for v in torch.autograd.grad([o, h], leaves, [do, dh])[:5]:
        assert v[:, (first // 64 + 1) * 64:].isfinite().all()
    # The other way round: a later document's NaN leaves the earlier one's chunks alone.
    ops2, _, do2, dh2 = make(1, 260, 1, 2, 40, 24, torch.float32)
    if what < 5:
        ops2[what][0, first + 5] = bad
    else:
        do2[0, first + 5] = bad
    leaves = [x.requires_grad_() for x in ops2]
    o, h = gated_delta(*leaves[:5], h0=leaves[5], reset=cut, return_state=True)
    hold("o", o[:, :first].detach(), good[0][:, :first].double(), REL)
    for v in torch.autograd.grad([o, h], leaves, [do2, dh2])[:5]:
        assert v[:, :first // 64 * 64].isfinite().all()


def test_gradients_against_differences():
    ops, cut, do, dh = make(1, 90, 1, 2, 12, 10, torch.float32, reset=0.03)
    leaves = [x.requires_grad_() for x in ops]
    o, h = gated_delta(*leaves[:5], h0=leaves[5], reset=cut, return_state=True)
    grads = torch.autograd.grad([o, h], leaves, [do, dh])
    step = 2.0 ** -8
    with torch.no_grad():
        for i, (v, grad) in enumerate(zip(leaves, grads)):
            way = torch.randn(v.shape, generator=torch.Generator(DEV).manual_seed(i), device=DEV)
            ends = []
            for sign in (1, -1):
                moved = [u + sign * step * way if u is v else u for u in leaves]
                oo, hh = gated_delta(*moved[:5], h0=moved[5], reset=cut, return_state=True)
                ends.append((oo.double() * do).sum() + (hh.double() * dh).sum())
            slope = (ends[0] - ends[1]) / (2 * step)
            along = (grad.double() * way).sum()
            # Third derivatives times step^2 / 6 = 2^-18.6 (of keys the chain of a hundred maps makes them
            # up to 2^11 times the slope), and the values' rounding over 2 step (2^-16 / 2^-7 of their size).
            size = (grad.double() * way).norm() + 2.0 ** -9 * (do.double().norm() + dh.double().norm())
            assert (slope - along).abs() <= 2e-2 * size, (i, slope, along)


def test_empty():
    for b, t in ((0, 5), (2, 0)):
        ops = [torch.empty(b, t, 1, 8, device=DEV) for _ in range(2)] + [torch.empty(b, t, 2, 4, device=DEV)]
        ops += [torch.empty(b, t, 2, device=DEV) for _ in range(2)] + [torch.ones(b, 2, 8, 4, device=DEV)]
        leaves = [x.requires_grad_() for x in ops]
        o, h = gated_delta(*leaves[:5], h0=leaves[5], return_state=True)
        assert o.shape == (b, t, 2, 4) and torch.equal(h, ops[5])
        got = torch.autograd.grad([o, h], leaves, [torch.ones_like(o), torch.ones_like(h)],
                                  allow_unused=True)
        assert (got[5] == 1).all()
        o, h = gated_delta(*ops[:5], return_state=True)
        assert (h == 0).all()


def test_mixed_types():
    ops, _, do, dh = make(2, 80, 1, 2, 24, 40, torch.float16)
    ops[2], ops[3], ops[4] = ops[2].float(), ops[3].bfloat16(), ops[4].float()
    ops[5] = ops[5].half()
    leaves = [x.requires_grad_() for x in ops]
    o, h = gated_delta(*leaves[:5], h0=leaves[5], return_state=True)
    assert o.dtype == torch.float32 and h.dtype == torch.float32
    ref = exact(ops, None, do.float(), dh)
    hold("o", o.detach(), ref["o"], REL)
    for name, v, got in zip(NAMES, leaves, torch.autograd.grad([o, h], leaves, [do.float(), dh])):
        assert got.dtype == v.dtype
        hold(name, got, ref[name], GRAD)


def everything(leaves, cut, do, dh):
    o, h = gated_delta(*leaves[:5], h0=leaves[5], reset=cut, return_state=True)
    return [o, h, *torch.autograd.grad([o, h], leaves, [do, dh])]


def test_repeats_bit_for_bit_and_on_other_streams():
    ops, cut, do, dh = make(2, 700, 2, 4, 128, 64, torch.bfloat16, reset=0.002)
    leaves = [x.requires_grad_() for x in ops]
    first = everything(leaves, cut, do, dh)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            other = everything(leaves, cut, do, dh)
    torch.cuda.current_stream().wait_stream(side)
    for u, v in zip(first, other):
        assert torch.equal(u, v)


def test_replays_in_a_graph():
    ops, cut, do, dh = make(2, 150, 1, 2, 40, 24, torch.float32, reset=0.01)
    leaves = [x.clone().requires_grad_() for x in ops]
    h = ops[5].clone()

    def once():
        return everything(leaves, cut, do, dh) + [gated_delta_step_(*(x[:, :1] for x in ops[:5]), h)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [v.detach() for v in once()]
    for rep in range(4):
        with torch.no_grad():
            leaves[2].copy_(torch.randn(ops[2].shape, generator=torch.Generator(DEV).manual_seed(rep),
                                        device=DEV))
        h.copy_(ops[5])
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in outs] + [h.clone()]
        h.copy_(ops[5])
        for u, v in zip(got, once() + [h]):
            assert torch.equal(u, v), rep


def test_compiles():
    ops, cut, do, dh = make(2, 100, 1, 2, 24, 20, torch.float32, reset=0.02)
    o, h = torch.ops.mambaqc.gated_delta(*ops, cut)
    leaves = [x.requires_grad_() for x in ops]
    o1, h1 = gated_delta(*leaves[:5], h0=leaves[5], reset=cut, return_state=True)
    assert torch.equal(o, o1) and torch.equal(h, h1)
    fn = lambda *x: gated_delta(*x[:5], h0=x[5], reset=cut, scale=0.5) * 2.0
    want = fn(*leaves)
    got = torch.compile(fn, backend="aot_eager", fullgraph=True)(*leaves)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, leaves, do), torch.autograd.grad(want, leaves, do)):
        assert torch.equal(a, b)


def test_step_tells_that_the_state_changed():
    ops, _, _, _ = make(2, 1, 1, 1, 8, 8, torch.float32)
    version = ops[5]._version
    gated_delta_step_(*ops)
    assert ops[5]._version > version


def test_second_and_forward_gradients_are_refused():
    ops, _, do, _ = make(2, 20, 1, 1, 8, 8, torch.float32)
    leaf = ops[2].requires_grad_()
    dv, = torch.autograd.grad(gated_delta(*ops[:5]), leaf, do, create_graph=True)
    with pytest.raises(RuntimeError, match="gradient of the gradient"):
        dv.sum().backward()
    ad = torch.autograd.forward_ad
    with ad.dual_level():
        dual = ad.make_dual(ops[0], torch.ones_like(ops[0]))
        with pytest.raises(RuntimeError):
            gated_delta(dual, *ops[1:5])


def copies(order):
    def pack(t):
        kept = torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)
        return kept if order == "dense" or t.dim() < 2 else kept.transpose(0, 1).contiguous().transpose(0, 1)
    return torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t)


@pytest.mark.parametrize("hooks", [lambda: copies("dense"), lambda: copies("turned"),
                                   torch.autograd.graph.save_on_cpu])
def test_saved_tensors_come_back_laid_out_anew(hooks):
    ops, cut, do, dh = make(3, 90, 2, 2, 24, 40, torch.bfloat16, reset=0.02)
    leaves = [x.requires_grad_() for x in ops]
    want = everything(leaves, cut, do, dh)
    with hooks():
        got = everything(leaves, cut, do, dh)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_registered_backward_checks_what_it_reads():
    ops, _, do, dh = make(2, 70, 1, 2, 24, 20, torch.float32)
    states, resid = torch.ops.mambaqc.gated_delta_train(*ops, None)[2:]
    op = torch.ops.mambaqc.gated_delta_backward
    op(*ops[:5], None, states, resid, do, dh)
    for bad in ((states[:, :1], resid, do, dh), (states, resid[:1], do, dh), (states, resid, do[:, :69], dh),
                (states, resid, do, dh[:1])):
        with pytest.raises(ValueError, match="must be"):
            op(*ops[:5], None, *bad)


def test_last_state_may_be_the_first():
    """The C entry point with h_last = h0."""
    import ctypes

    ops, _, _, _ = make(2, 100, 2, 2, 40, 24, torch.float32)
    want, last = gated_delta(*ops[:5], h0=ops[5], return_state=True)
    o, h = torch.empty_like(ops[2]), ops[5].clone()
    nbytes = nat.load().mqc_gated_delta_workspace_bytes(2, 100, 2, 2, 40, 24, 0, 0)
    ws = torch.empty(nbytes, device=DEV, dtype=torch.uint8)
    strides = (ctypes.c_int64 * 9)(*(s for x in ops[:3] for s in x.stride()[:3]))
    nat.call("mqc_gated_delta_fwd", o, *(x.data_ptr() for x in ops[:3]), strides, ops[3].data_ptr(), 0,
             ops[4].data_ptr(), 0, None, h.data_ptr(), o.data_ptr(), h.data_ptr(), None, None, 2, 100, 2, 2,
             40, 24, 40 ** -0.5, 0, ws.data_ptr(), nbytes, nat.stream_of(o))
    assert torch.equal(o, want) and torch.equal(h, last)


def test_offsets_past_32_bits():
    """Tokens more than 2^32 elements apart, read in place."""
    ops, _, do, dh = make(1, 3, 1, 1, 32, 32, torch.bfloat16)
    far = torch.empty((1 << 32) + 4096, device=DEV, dtype=torch.bfloat16)
    views = [far[1000 * i:].as_strided((1, 3, 1, 32), (0, 1 << 31, 32, 1)) for i in range(3)]
    for view, x in zip(views, ops[:3]):
        view.copy_(x)
    want = gated_delta(*ops[:5])
    assert torch.equal(gated_delta(*views, *ops[3:5]), want)


def test_many_tokens_past_32_bit_offsets():
    """A sequence whose outputs and workspace pass 2^32 bytes: its end, behind a reset, alone."""
    t, tail = 300_000, 200
    gen = torch.Generator(DEV).manual_seed(3)
    qk = torch.randn(1, t, 2, 64, generator=gen, device=DEV, dtype=torch.bfloat16)
    qk /= qk.float().norm(dim=-1, keepdim=True).bfloat16()
    v = torch.randn(1, t, 64, 128, generator=gen, device=DEV, dtype=torch.bfloat16)
    g, beta = torch.full((1, t, 64), -0.05, device=DEV), torch.full((1, t, 64), 0.5, device=DEV)
    cut = torch.zeros(1, t, dtype=torch.bool, device=DEV)
    cut[0, t - tail] = True
    q, k = qk[:, :, :1], qk[:, :, 1:]
    o, h = gated_delta(q, k, v, g, beta, reset=cut, return_state=True)
    o1, h1 = gated_delta(*(x[:, t - tail:] for x in (q, k, v, g, beta)), return_state=True)
    hold("o", o[:, t - tail:], o1.double(), REL + torch.finfo(torch.bfloat16).eps)
    hold("h", h, h1.double(), REL)


# Beyond 256 tiles of 16 columns two workgroups share a CU, beyond 512 one has two tiles.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch", [4, 7])
@pytest.mark.parametrize("dk", [20, 60, 128])
def test_many_heads(dtype, batch, dk):
    check(*make(batch, 150, 8, 16, dk, 70, dtype, reset=0.02))


@pytest.mark.parametrize("batch", [70, 140])
@pytest.mark.parametrize("what", range(5))
def test_nan_stays_before_a_reset_with_many_heads(batch, what):
    ops, _, do, dh = make(batch, 150, 1, 2, 40, 24, torch.float32)
    cut = torch.zeros(batch, 150, dtype=torch.bool, device=DEV)
    cut[:, 40] = True
    good = gated_delta(*ops[:5], h0=ops[5], reset=cut, return_state=True)
    ops[what][::3, 20, ..., 0] = float("nan")
    leaves = [x.requires_grad_() for x in ops]
    o, h = gated_delta(*leaves[:5], h0=leaves[5], reset=cut, return_state=True)
    hold("o", o[:, 40:].detach(), good[0][:, 40:].double(), REL)
    hold("h", h.detach(), good[1].double(), REL)
    for v in torch.autograd.grad([o, h], leaves, [do, dh])[:5]:
        assert v[:, 64:].isfinite().all() and v[1::3].isfinite().all()


@pytest.mark.parametrize("dk", [24, 100])
def test_what_nothing_decays_into_has_no_gradient(dk):
    """log_decay of the first token without a state, of a document's first one and where the state is zero."""
    ops, _, do, dh = make(2, 140, 1, 2, dk, 40, torch.float32, h0=False)
    cut = torch.zeros(2, 140, dtype=torch.bool, device=DEV)
    cut[0, [5, 64, 100]] = True
    g = ops[3].requires_grad_()
    for reset, h0 in ((None, None), (cut, None), (cut, torch.zeros(2, 2, dk, 40, device=DEV))):
        o, h = gated_delta(*ops[:5], h0=h0, reset=reset, return_state=True)
        got, = torch.autograd.grad([o, h], g, [do, dh])
        assert (got[:, 0] == 0).all() and (got[:, 1:4] != 0).any()
        if reset is not None:
            assert (got[cut] == 0).all()
    with torch.no_grad():
        ops[2][:, :64] = 0  # nothing is written in the first chunk
    o, h = gated_delta(*ops[:5], return_state=True)
    assert (torch.autograd.grad([o, h], g, [do, dh])[0][:, 64] == 0).all()


RATES = (0.5, 5.0, 10.0, 15.0, 30.0, 80.0, 200.0, 1e5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dk,reset", [(24, 0.0), (60, 0.03), (101, 0.02), (128, 0.0), (128, 0.03)])
def test_gradient_of_log_decay_of_heads_that_forget_fast(dtype, dk, reset):
    """Every term of log_decay's gradient has its token's factor exp(log_decay), so a head's gradients are as
    small as that, and held to a head's own size. (The exponent of a factor is an fp32 number: of the largest
    one that is not zero, 87, half a step is 2^-18 of the factor.) Where a factor is 0, so is the gradient."""
    ops, cut, do, dh = make(1, 200, 4, 8, dk, 40, dtype, reset=reset)
    for head, rate in enumerate(RATES):
        ops[3][:, :, head] = -rate
    ref = [x.clone() for x in ops]
    ref[3] = ops[3].clamp_min(-700.0)  # exp of it is 0 to 64 bits too, and its slope a number
    want = exact(ref, cut, do, dh)["g"]
    leaves = [x.detach().requires_grad_() for x in ops]
    o, h = gated_delta(*leaves[:5], h0=leaves[5], reset=cut, return_state=True)
    got, = torch.autograd.grad([o, h], leaves[3], [do, dh])
    for head, rate in enumerate(RATES):
        hold(rate, got[..., head], want[..., head], GRAD)
        assert rate < 104 or (got[..., head] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dk", [24, 60, 128])
def test_gradient_of_log_decay_of_tokens_that_forget(dtype, dk):
    """Single tokens that forget much or all, among ones that forget little: each held to its own gradient, in
    terms of the size that its factor gives it."""
    ops, _, do, dh = make(2, 150, 2, 2, dk, 40, dtype, rate=0.02)
    for at, rate in ((7, 12.0), (40, 20.0), (64, 16.0), (127, 25.0), (149, 14.0)):
        ops[3][:, at] = -rate
    want = exact(ops, None, do, dh)["g"]
    leaves = [x.detach().requires_grad_() for x in ops]
    o, h = gated_delta(*leaves[:5], h0=leaves[5], return_state=True)
    got, = torch.autograd.grad([o, h], leaves[3], [do, dh])
    # Without its factor a token's gradient is of the size that the other tokens' are.
    size = want.square().mean().sqrt() * ops[3].double().exp()
    off = (got.double() - want).abs()
    assert (off <= 2.0 ** -24 * want.abs() + GRAD * torch.maximum(want.abs(), 8 * size)).all(), (off / size).max()
