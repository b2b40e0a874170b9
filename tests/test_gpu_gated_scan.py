"""The gated scan (csrc/gated_scan.hip) against the recurrence walked in 64 bits: values, states and
gradients at sizes around its chunks and tiles, resets, strides, states, the single-token step, slow
channels, NaN behind a reset, other streams and graphs.

Tolerances. The kernels' gates carry a relative error of a few 2^-24 each (the exponentials' own and
the rounding of their arguments, up to 2^-20 together for |dt| up to 8), the sums are convex, so a
result is off by at most 2^-18 of the same expression with every term taken by its absolute value
(`mag`), twice that for a product of two such results, plus half a step of its type.
"""
import pytest
import torch

from mambaqc_amd.kernels import gated_scan, gated_scan_step_

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
REL = 2.0 ** -18


def walk(dt, g, x, lam, h0, reset, dy=None, dh=None):
    """Values, gradients and their magnitudes, in 64 bits, token by token."""
    dt, g, x, lam = (v.detach().double() for v in (dt, g, x, lam))
    b, t, d = x.shape
    p = torch.nn.functional.softplus(dt, threshold=100) * lam.exp()
    a, w, sig = (-p).exp(), -torch.expm1(-p), torch.sigmoid(g)
    s = sig * x
    keep = a if reset is None else torch.where(reset[..., None], 0.0, a)
    h = x.new_zeros(b, d) if h0 is None else h0.double()
    hm = h.abs()
    prev, prevm, hs, hms = [], [], [], []
    for i in range(t):
        dead = torch.zeros(b, 1, dtype=torch.bool, device=x.device) if reset is None \
            else reset[:, i, None]
        h, hm = torch.where(dead, 0.0, h), torch.where(dead, 0.0, hm)
        prev.append(h)
        prevm.append(hm)
        h, hm = a[:, i] * h + w[:, i] * s[:, i], a[:, i] * hm + w[:, i] * s[:, i].abs()
        hs.append(h)
        hms.append(hm)
    empty = x.new_empty(b, 0, d)
    stack = lambda v: torch.stack(v, 1) if v else empty
    out = {"y": (stack(hs), stack(hms)), "h": (h, hm)}
    if dy is None:
        return out
    prev, prevm = stack(prev), stack(prevm)
    G, Gm = torch.empty_like(x), torch.empty_like(x)
    acc = x.new_zeros(b, d) if dh is None else dh.double()
    accm = acc.abs()
    for i in reversed(range(t)):
        acc, accm = acc + dy[:, i].double(), accm + dy[:, i].double().abs()
        G[:, i], Gm[:, i] = acc, accm
        acc, accm = acc * a[:, i], accm * a[:, i]
        if reset is not None:
            acc = torch.where(reset[:, i, None], 0.0, acc)
            accm = torch.where(reset[:, i, None], 0.0, accm)
    dp, dpm = a * G * (s - prev), a * Gm * (s.abs() + prevm)
    sd = torch.sigmoid(dt) * lam.exp()
    out |= {"dt": (dp * sd, 2 * dpm * sd), "g": (w * G * s * (1 - sig), 2 * w * Gm * s.abs() * (1 - sig)),
            "x": (w * G * sig, w * Gm * sig), "rate": ((dp * p).sum((0, 1)), 4 * (dpm * p).sum((0, 1))),
            "h0": (acc, accm)}
    return out


def hold(what, got, ref):
    want, mag = ref
    half = torch.finfo(got.dtype).eps / 2
    off = (got.double() - want).abs()
    assert got.shape == want.shape, what
    bad = ~(off <= half * want.abs() + REL * mag + torch.finfo(got.dtype).tiny)
    assert not bad.any(), (what, int(bad.sum()), off[bad][:4], want[bad][:4], mag[bad][:4])


def make(b, t, d, dtype, seed=0, h0=True, reset=0.0, slow=False):
    gen = torch.Generator(device=DEV).manual_seed(seed + 7 * b + 11 * t + 13 * d)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    dt, g, x = (r(b, t, d) * 1.5 - 1).to(dtype), r(b, t, d).to(dtype), r(b, t, d).to(dtype)
    lam = torch.rand(d, generator=gen, device=DEV) * 7.6 - 6.9
    cut = torch.rand(b, t, generator=gen, device=DEV) < reset if reset else None
    return dt, g, x, lam, r(b, d) if h0 else None, cut, r(b, t, d).to(dtype), r(b, d)


# Around a chunk of 32 steps and the tiles of 64 channels, and longer walks; odd widths.
SIZES = [(1, 1, 1), (2, 2, 3), (1, 31, 64), (3, 32, 65), (1, 33, 130), (2, 64, 8), (1, 129, 258),
         (2, 257, 100), (1, 1000, 36), (2, 1031, 7), (1, 4100, 66)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,t,d", SIZES)
@pytest.mark.parametrize("state,reset", [(False, 0.0), (True, 0.05)])
def test_values_and_gradients(dtype, b, t, d, state, reset):
    dt, g, x, lam, h0, cut, dy, dh = make(b, t, d, dtype, h0=state, reset=reset)
    ref = walk(dt, g, x, lam, h0, cut, dy, dh)
    with torch.no_grad():
        y0, h = gated_scan(dt, g, x, lam, h0=h0, reset=cut, return_state=True)
    hold("y", y0, ref["y"])
    hold("h", h, ref["h"])
    names = ["dt", "g", "x", "rate"] + (["h0"] if state else [])
    leaves = [v.requires_grad_() for v in (dt, g, x, lam)] + ([h0.requires_grad_()] if state else [])
    y, h = gated_scan(dt, g, x, lam, h0=h0, reset=cut, return_state=True)
    assert torch.equal(y, y0)
    for name, got in zip(names, torch.autograd.grad([y, h], leaves, [dy, dh])):
        hold(name, got, ref[name])


@pytest.mark.parametrize("which", ["y", "h"])
def test_one_output_alone(which):
    dt, g, x, lam, h0, _, dy, dh = make(2, 70, 20, torch.float32)
    leaves = [v.requires_grad_() for v in (dt, g, x, lam, h0)]
    y, h = gated_scan(*leaves[:4], h0=h0, return_state=True)
    ref = walk(dt, g, x, lam, h0, None, dy if which == "y" else torch.zeros_like(dy),
               dh if which == "h" else None)
    got = torch.autograd.grad(y if which == "y" else h, leaves, dy if which == "y" else dh)
    for name, v in zip(["dt", "g", "x", "rate", "h0"], got):
        hold(name, v, ref[name])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 48, 33])
def test_views_are_read_in_place(dtype, d):
    """Parts of one projection's output, whose tokens are 3 d and more apart, and a transposed one."""
    wide = torch.randn(2, 50, 3 * d + 5, device=DEV).to(dtype)
    dt, g, x = wide[..., :d], wide[..., d:2 * d], wide[..., 2 * d + 5:]
    lam, dy = torch.randn(d, device=DEV) - 2, torch.randn(2, 50, d, device=DEV).to(dtype)
    ref = walk(dt, g, x, lam, None, None, dy)
    leaves = [v.detach().requires_grad_() for v in (dt, g, x, lam)]
    y = gated_scan(*leaves)
    hold("y", y, ref["y"])
    for name, got in zip(["dt", "g", "x", "rate"],
                         torch.autograd.grad(y, leaves, dy.transpose(0, 1).contiguous().transpose(0, 1))):
        hold(name, got, ref[name])
    turned = [v.transpose(1, 2).contiguous().transpose(1, 2) for v in (dt, g, x)]
    assert torch.equal(gated_scan(*turned, lam), y)
    # One token for every sequence, batches apart as in a longer buffer; and a broadcast batch.
    hold("y", gated_scan(dt[:, 7:8], g[:, 7:8], x[:, 7:8], lam),
         walk(dt[:, 7:8], g[:, 7:8], x[:, 7:8], lam, None, None)["y"])
    one = [v[:1].expand(2, -1, -1) for v in (dt, g, x)]
    assert torch.equal(gated_scan(*one, lam)[1], y[0])
    leaf = x[:1].detach().requires_grad_()
    y2 = gated_scan(one[0], one[1], leaf.expand(2, -1, -1), lam)
    hold("x", torch.autograd.grad(y2, leaf, dy)[0].float(),
         tuple(sum(v[i:i + 1] for i in range(2)) * k for v, k in zip(
             walk(*one, lam, None, None, dy)["x"], (1, 1 + 2 * torch.finfo(dtype).eps / REL))))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,d", [(1, 1), (4, 1536), (16, 130), (3, 257)])
def test_step(dtype, b, d):
    """Twenty steps, each equal to the whole walk's token to the gates' error."""
    dt, g, x, lam, h0, _, _, _ = make(b, 20, d, dtype)
    ref = walk(dt, g, x, lam, h0, None)
    h = h0.clone()
    for i in range(20):
        y = gated_scan_step_(dt[:, i:i + 1], g[:, i:i + 1], x[:, i:i + 1], lam, h)
        hold("y", y[:, 0], tuple(v[:, i] for v in ref["y"]))
    hold("h", h, ref["h"])


def test_state_continues_a_split_sequence():
    dt, g, x, lam, h0, cut, _, _ = make(2, 300, 40, torch.float32, reset=0.02)
    whole, h = gated_scan(dt, g, x, lam, h0=h0, reset=cut, return_state=True)
    at, parts = h0, []
    for lo, hi in ((0, 1), (1, 1), (1, 97), (97, 300)):
        y, at = gated_scan(dt[:, lo:hi], g[:, lo:hi], x[:, lo:hi], lam, h0=at,
                           reset=cut[:, lo:hi], return_state=True)
        parts.append(y)
    ref = walk(dt, g, x, lam, h0, cut)
    hold("y", torch.cat(parts, 1), ref["y"])
    hold("h", at, ref["h"])
    hold("h", h, ref["h"])


def test_slow_channels_keep_their_gain():
    """Constant input, channels that hold for up to 2e6 tokens: the state goes to (1 - e^{-rate D t}) s.
    A decay rounded to fp32 would be off by 2^-25 of the state at each token, the same way each time."""
    t, d = 20000, 64
    dt = torch.full((1, t, d), 0.3, device=DEV)
    g, x = torch.full_like(dt, 40.0), torch.ones_like(dt)
    lam = torch.linspace(-14, -1, d, device=DEV)
    y, h = gated_scan(dt, g, x, lam, return_state=True)
    delta = torch.nn.functional.softplus(dt.double()) * lam.double().exp()
    want = -torch.expm1(-delta.cumsum(1))
    # Each token rounds the state once: at most t / 2 steps of 2^-24 against a state that grows over
    # those tokens; rounding goes both ways, and sqrt(t) of them is what is left (141 at 20000).
    assert ((y.double() - want).abs() <= 141 * 2.0 ** -24 * want + 2.0 ** -20 * want).all()


@pytest.mark.parametrize("t", [40, 700])
def test_nan_and_inf_stay_before_a_reset(t):
    dt, g, x, lam, h0, _, dy, dh = make(2, t, 30, torch.float32)
    cut = torch.zeros(2, t, dtype=torch.bool, device=DEV)
    at = t // 2 + 3
    cut[:, at] = True
    h0[0, :5] = float("nan")
    h0[1, 3] = float("inf")
    x[0, at - 1, 7] = float("nan")
    x[1, 2, 9] = float("inf")
    ref = walk(dt, g, x, lam, h0, cut, dy, dh)
    leaves = [v.requires_grad_() for v in (dt, g, x)]
    y, h = gated_scan(*leaves, lam, h0=h0, reset=cut, return_state=True)
    assert torch.isfinite(y[:, at:]).all() and torch.isfinite(h).all()
    assert torch.isnan(y[0, at - 1, 7]) and torch.isnan(y[0, 0, :5]).all()
    hold("y", y[:, at:].detach(), tuple(v[:, at:] for v in ref["y"]))
    for name, got in zip(["dt", "g", "x"], torch.autograd.grad([y, h], leaves, [dy, dh])):
        hold(name, got[:, at:], tuple(v[:, at:] for v in ref[name]))
    # A NaN in the gradient behind the reset does not go before it.
    bad = dy.clone()
    bad[:, at + 1] = float("nan")
    y = gated_scan(*leaves, lam, reset=cut)
    assert torch.isfinite(torch.autograd.grad(y, leaves[2], bad)[0][:, :at]).all()


def test_extreme_gates():
    """dt and g at the ends of their types: gates of exactly 0 and 1, no NaN."""
    big = torch.tensor([-1e4, -200.0, -90.0, 0.0, 90.0, 200.0, 1e4], device=DEV)
    dt, g = (v.reshape(1, -1, 1).repeat(1, 1, 4) for v in torch.meshgrid(big, big, indexing="ij"))
    x, lam = torch.ones_like(dt), torch.tensor([-20.0, 0.0, 5.0, 80.0], device=DEV)
    dy = torch.ones_like(x)
    leaves = [v.requires_grad_() for v in (dt, g, x, lam)]
    y = gated_scan(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    ref = walk(dt, g, x, lam, None, None, dy)
    hold("y", y, ref["y"])
    for v in grads:
        assert torch.isfinite(v).all()
    hold("x", grads[2], ref["x"])


def test_gradients_against_differences():
    dt, g, x, lam, h0, cut, dy, dh = make(1, 90, 6, torch.float32, reset=0.03)
    leaves = [v.requires_grad_() for v in (dt, g, x, lam, h0)]
    y, h = gated_scan(*leaves[:4], h0=h0, reset=cut, return_state=True)
    grads = torch.autograd.grad([y, h], leaves, [dy, dh])
    step = 2.0 ** -6
    with torch.no_grad():
        for i, (v, grad) in enumerate(zip(leaves, grads)):
            way = torch.randn(v.shape, generator=torch.Generator(DEV).manual_seed(i), device=DEV)
            ends = []
            for sign in (1, -1):
                moved = [u + sign * step * way if u is v else u for u in leaves]
                yy, hh = gated_scan(*moved[:4], h0=moved[4], reset=cut, return_state=True)
                ends.append((yy.double() * dy).sum() + (hh.double() * dh).sum())
            slope = (ends[0] - ends[1]) / (2 * step)
            along = (grad.double() * way).sum()
            # Third derivatives times step^2 / 6 (4e-5 of gates' slopes), and the values' rounding
            # over 2 step (2^-18 / 2^-5 of their size).
            size = (grad.double() * way).norm() + 2.0 ** -13 * (dy.double().norm() + dh.double().norm())
            assert (slope - along).abs() <= 2e-2 * size, (i, slope, along)


def test_empty():
    e = lambda *s: torch.empty(*s, device=DEV, requires_grad=True)
    for b, t, d in ((0, 5, 8), (2, 0, 8), (2, 5, 0)):
        leaves = [e(b, t, d) for _ in range(3)]
        lam = torch.zeros(d, device=DEV, requires_grad=True)
        h0 = torch.ones(b, d, device=DEV, requires_grad=True)
        y, h = gated_scan(*leaves, lam, h0=h0, return_state=True)
        assert y.shape == (b, t, d) and h.shape == (b, d)
        if t == 0:
            assert torch.equal(h, h0)
        got = torch.autograd.grad([y, h], leaves + [lam, h0], [torch.ones_like(y), torch.ones_like(h)],
                                  allow_unused=True)
        assert (got[3] == 0).all()
        if t == 0:
            assert (got[4] == 1).all()


def test_mixed_types_and_parameters():
    dt, g, x, lam, h0, _, dy, _ = make(2, 40, 24, torch.float16)
    x = x.float()
    leaves = [dt.requires_grad_(), g.requires_grad_(), x.requires_grad_(),
              lam.bfloat16().requires_grad_(), h0.half().requires_grad_()]
    y = gated_scan(*leaves[:4], h0=leaves[4])
    assert y.dtype == torch.float32
    ref = walk(dt, g, x, leaves[3], leaves[4].detach().float(), None, dy.float())
    hold("y", y, ref["y"])
    for name, v, got in zip(["dt", "g", "x", "rate", "h0"], leaves,
                            torch.autograd.grad(y, leaves, dy.float())):
        assert got.dtype == v.dtype
        hold(name, got, ref[name])


def test_repeats_bit_for_bit_and_on_other_streams():
    dt, g, x, lam, h0, cut, dy, dh = make(2, 3000, 192, torch.bfloat16, reset=0.002)
    leaves = [v.requires_grad_() for v in (dt, g, x, lam, h0)]

    def once():
        y, h = gated_scan(*leaves[:4], h0=h0, reset=cut, return_state=True)
        return [y, h, *torch.autograd.grad([y, h], leaves, [dy, dh])]

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            other = once()
    torch.cuda.current_stream().wait_stream(side)
    for u, v in zip(first, other):
        assert torch.equal(u, v)


def test_replays_in_a_graph():
    dt, g, x, lam, h0, cut, dy, dh = make(2, 500, 96, torch.float32, reset=0.01)
    leaves = [v.clone().requires_grad_() for v in (dt, g, x, lam, h0)]
    h = h0.clone()

    def once():
        y, hl = gated_scan(*leaves[:4], h0=leaves[4], reset=cut, return_state=True)
        return [y, hl, *torch.autograd.grad([y, hl], leaves, [dy, dh]),
                gated_scan_step_(dt[:, :1], g[:, :1], x[:, :1], lam, h)]

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
            leaves[2].copy_(torch.randn(x.shape, generator=torch.Generator(DEV).manual_seed(rep),
                                        device=DEV))
        h.copy_(h0)
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in outs]
        h.copy_(h0)
        for u, v in zip(got, once()):
            assert torch.equal(u, v), rep


def test_compiled_operators():
    """torch.ops.mambaqc.gated_scan and gated_scan_train, and their gradient."""
    dt, g, x, lam, h0, cut, dy, _ = make(2, 50, 16, torch.float32, reset=0.05)
    y, h = torch.ops.mambaqc.gated_scan(dt, g, x, lam, h0, cut)
    leaves = [v.requires_grad_() for v in (dt, g, x, lam, h0)]
    y1, h1 = gated_scan(*leaves[:4], h0=h0, reset=cut, return_state=True)
    assert torch.equal(y, y1) and torch.equal(h, h1)
    y2 = torch.ops.mambaqc.gated_scan_train(*leaves, cut)[0]
    for u, v in zip(torch.autograd.grad(y2, leaves, dy), torch.autograd.grad(y1, leaves, dy)):
        assert torch.equal(u, v)


# The spans, chunks and groups of chunks that the walks are cut into (forward 16, 128 and 2048 steps,
# backward 16, 64 and 1024), each one short, full and one over.
@pytest.mark.parametrize("t", [15, 16, 17, 63, 64, 65, 127, 128, 1023, 1024, 1025, 2047, 2048, 2049, 5000])
@pytest.mark.parametrize("reset", [0.0, 0.01])
def test_around_spans_chunks_and_groups(t, reset):
    dt, g, x, lam, h0, cut, dy, dh = make(2, t, 37, torch.float32, reset=reset)
    ref = walk(dt, g, x, lam, h0, cut, dy, dh)
    leaves = [v.requires_grad_() for v in (dt, g, x, lam, h0)]
    y, h = gated_scan(*leaves[:4], h0=h0, reset=cut, return_state=True)
    hold("y", y, ref["y"])
    hold("h", h, ref["h"])
    for name, got in zip(["dt", "g", "x", "rate", "h0"], torch.autograd.grad([y, h], leaves, [dy, dh])):
        hold(name, got, ref[name])


@pytest.mark.parametrize("at", [0, 15, 16, 63, 64, 127, 128, 2047, 2048])
def test_reset_at_the_ends_of_chunks(at):
    dt, g, x, lam, h0, _, dy, dh = make(1, 2200, 66, torch.float32)
    cut = torch.zeros(1, 2200, dtype=torch.bool, device=DEV)
    cut[0, at] = True
    ref = walk(dt, g, x, lam, h0, cut, dy, dh)
    leaves = [v.requires_grad_() for v in (dt, g, x, lam, h0)]
    y, h = gated_scan(*leaves[:4], h0=h0, reset=cut, return_state=True)
    hold("y", y, ref["y"])
    for name, got in zip(["dt", "g", "x", "rate", "h0"], torch.autograd.grad([y, h], leaves, [dy, dh])):
        hold(name, got, ref[name])


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_nan_goes_through_all_chunks(bad):
    """States that are not finite pass from chunk to chunk like others, in their channel alone."""
    dt, g, x, lam, h0, _, dy, dh = make(1, 4500, 70, torch.float32)
    x[0, 130, 9] = bad
    leaves = [v.requires_grad_() for v in (dt, g, x)]
    y, h = gated_scan(*leaves, lam, h0=h0, return_state=True)
    others = [i for i in range(70) if i != 9]
    assert not y[0, 130:, 9].isfinite().any() and y[0, :130].isfinite().all()
    assert y[0][:, others].isfinite().all() and not h[0, 9].isfinite()
    dy[0, 4000, 11] = bad
    for v in torch.autograd.grad([y, h], leaves, [dy, dh]):
        assert v[0][:, [i for i in others if i != 11]].isfinite().all()
        assert v[0, 4001:, 11].isfinite().all() and not v[0, 3999, 11].isfinite()


def test_last_state_may_be_the_first():
    """The C entry point with h_last = h0, over several chunks and within one."""
    from mambaqc_amd import _native as nat

    for t in (1, 100, 2500):
        dt, g, x, lam, h0, _, _, _ = make(2, t, 100, torch.float32)
        ref = walk(dt, g, x, lam, h0, None)
        y, h = torch.empty_like(x), h0.clone()
        nbytes = nat.load().mqc_gated_scan_workspace_bytes(2, t, 100)
        ws = torch.empty(nbytes, device=DEV, dtype=torch.uint8)
        nat.call("mqc_gated_scan_fwd", x, dt.data_ptr(), 100, g.data_ptr(), 100, x.data_ptr(), 100,
                 lam.data_ptr(), h.data_ptr(), None, y.data_ptr(), h.data_ptr(), None, 2, t, 100, 0,
                 ws.data_ptr(), nbytes, nat.stream_of(x))
        hold("y", y, ref["y"])
        hold("h", h, ref["h"])


def test_fast_channels_underflow_cleanly():
    """Gradients that reach back through decays of 2^-100 and less of a state: exact to the gates' error,
    then 0, and never NaN."""
    t, d = 300, 64
    dt = torch.zeros(1, t, d, device=DEV)
    g, x = torch.zeros_like(dt), torch.ones_like(dt)
    lam = torch.linspace(-3, 12, d, device=DEV)
    leaves = [v.requires_grad_() for v in (dt, g, x, lam)]
    y, h = gated_scan(*leaves, return_state=True)
    dh = torch.ones(1, d, device=DEV)
    ref = walk(dt, g, x, lam, None, None, torch.zeros_like(x), dh)
    for name, got in zip(["dt", "g", "x", "rate"], torch.autograd.grad(h, leaves, dh)):
        assert got.isfinite().all()
        want, mag = ref[name]
        # A decay over n steps carries n gates' errors (2^-21 each) of its own.
        n = torch.arange(t, 0, -1, device=DEV)[None, :, None] if got.dim() == 3 else t
        assert ((got.double() - want).abs() <= (REL + n * 2.0 ** -21) * mag + 1e-37).all(), name


def test_second_gradients_are_refused():
    dt, g, x, lam, _, _, dy, _ = make(1, 20, 8, torch.float32)
    x.requires_grad_()
    dx, = torch.autograd.grad(gated_scan(dt, g, x, lam), x, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="gradient of the gradient"):
        dx.sum().backward()


def test_offsets_past_32_bits():
    """Rows more than 2^32 bytes into their tensors, read in place and written: what lies behind a reset
    near the end equals that part alone (another cut into spans: each gate's error, not the same bits)."""
    t, d, tail = 1_100_000, 1024, 700
    wide = torch.empty(1, t, 3 * d, device=DEV, dtype=torch.bfloat16).normal_()
    dt, g, x = wide.split(d, -1)
    lam = torch.linspace(-6, 0, d, device=DEV)
    cut = torch.zeros(1, t, dtype=torch.bool, device=DEV)
    cut[0, t - tail] = True
    end = [v[:, t - tail:].clone().requires_grad_() for v in (dt, g, x)]
    leaves = [v.detach().requires_grad_() for v in (dt, g, x)]
    y, h = gated_scan(*leaves, lam, reset=cut, return_state=True)
    y1, h1 = gated_scan(*end, lam, return_state=True)
    ref = walk(*end, lam, None, None, dy := torch.randn_like(y1), torch.ones_like(h1))
    hold("y", y[:, t - tail:].detach(), ref["y"])
    hold("h", h.detach(), ref["h"])
    whole = torch.zeros_like(y)
    whole[:, t - tail:] = dy
    for name, got in zip(("dt", "g", "x"), torch.autograd.grad([y, h], leaves, [whole, torch.ones_like(h)])):
        hold(name, got[:, t - tail:], ref[name])
        assert (got[:, :t - tail] == 0).all()


def test_compiles():
    """Traced through the registered operators, with the same results."""
    dt, g, x, lam, h0, cut, dy, _ = make(2, 150, 24, torch.float32, reset=0.02)
    leaves = [v.requires_grad_() for v in (dt, g, x, lam, h0)]
    fn = lambda *v: gated_scan(*v[:4], h0=v[4], reset=cut) * 2.0
    want = fn(*leaves)
    got = torch.compile(fn, backend="aot_eager", fullgraph=True)(*leaves)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, leaves, dy), torch.autograd.grad(want, leaves, dy)):
        assert torch.equal(a, b)


def test_step_tells_that_the_state_changed():
    dt, g, x, lam, h0, _, _, _ = make(2, 1, 24, torch.float32)
    version = h0._version
    gated_scan_step_(dt, g, x, lam, h0)
    assert h0._version > version


@pytest.mark.parametrize("dtype,shape", [(torch.bfloat16, (1, 7000, 4100)), (torch.bfloat16, (1, 9000, 4100)),
                                         (torch.bfloat16, (2, 8209, 4100)), (torch.float32, (1, 7000, 2050)),
                                         (torch.float32, (3, 5000, 2050))])
def test_sizes_past_the_cache_equal_their_parts(dtype, shape):
    """Operands past 256 MiB, in all, in the inputs alone or in neither: channel by channel the same
    bits as a few channels at a time, gradients too."""
    gen = torch.Generator(DEV).manual_seed(8)
    full = [torch.randn(shape, generator=gen, device=DEV, dtype=dtype).requires_grad_() for _ in range(3)]
    rate = (torch.rand(shape[2], generator=gen, device=DEV) * -4).requires_grad_()
    dy = torch.randn(shape, generator=gen, device=DEV, dtype=dtype)
    y, h = gated_scan(*full, rate, return_state=True)
    grads = torch.autograd.grad((y, h), [*full, rate], (dy, torch.ones_like(h)))
    for start in range(0, shape[2], 1024):
        part = slice(start, start + 1024)
        leaves = [t.detach()[..., part].contiguous().requires_grad_() for t in (*full, rate)]
        some, last = gated_scan(*leaves, return_state=True)
        want = torch.autograd.grad((some, last), leaves, (dy[..., part], torch.ones_like(last)))
        assert torch.equal(y[..., part], some) and torch.equal(h[..., part], last)
        assert all(torch.equal(g[..., part], w) for g, w in zip(grads, want))


def copies(order):
    """Hooks on saved tensors that give back dense copies, or ones whose axes lie in another order."""
    def pack(t):
        kept = torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)
        return kept if order == "dense" or t.dim() < 2 else kept.transpose(0, 1).contiguous().transpose(0, 1)
    return torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t)


@pytest.mark.parametrize("hooks", [lambda: copies("dense"), lambda: copies("turned"),
                                   torch.autograd.graph.save_on_cpu])
@pytest.mark.parametrize("t", [1, 40, 300])
def test_saved_tensors_come_back_laid_out_anew(hooks, t):
    """The backward reads what hooks on saved tensors give back, not the forward's rows."""
    wide = torch.randn(3, t, 5 * 24, generator=torch.Generator(DEV).manual_seed(t), device=DEV)
    cut = torch.arange(3 * t, device=DEV).reshape(3, t) % 37 == 5
    dy = torch.randn(3, t, 24, device=DEV)

    def grads():
        leaf = wide.detach().requires_grad_()
        lam = torch.linspace(-4, 1, 24, device=DEV).requires_grad_()
        y, h = gated_scan(leaf[..., 24:48], leaf[..., 48:72], leaf[..., 96:], lam, reset=cut,
                          return_state=True)
        return torch.autograd.grad([y, h], [leaf, lam], [dy, torch.ones_like(h)])

    want = grads()
    with hooks():
        got = grads()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_saved_tensors_of_other_shapes_are_refused():
    dt, g, x, lam, _, _, dy, _ = make(2, 70, 24, torch.float32)
    x.requires_grad_()
    for shape in [(2, 70, 24), (24,), (2, 2, 24)]:
        with torch.autograd.graph.saved_tensors_hooks(
                lambda t: t, lambda t: t[:1] if tuple(t.shape) == shape else t):
            y = gated_scan(dt, g, x, lam)
        with pytest.raises(ValueError, match="must be|other shapes"):
            y.backward(dy)


def test_registered_backward_checks_what_it_reads():
    dt, g, x, lam, _, _, dy, dh = make(2, 70, 24, torch.float32)
    carries = torch.ops.mambaqc.gated_scan_train(dt, g, x, lam, None, None)[2]
    op = torch.ops.mambaqc.gated_scan_backward
    op(dt, g, x, lam, None, carries, dy, dh)
    for bad in ((carries[:, :1], dy, dh), (carries, dy[:, :69], dh), (carries, dy, dh[:1])):
        with pytest.raises(ValueError, match="must be"):
            op(dt, g, x, lam, None, *bad)
    with pytest.raises(RuntimeError, match="ROCm device"):
        op(dt, g, x, lam, None, carries.cpu(), dy, dh)


def hold_kinds(what, got, ref):
    """hold() where the reference is finite; the same infinities, and nothing finite for a NaN."""
    want, mag = ref
    fine, inf = want.isfinite(), want.isinf()
    assert torch.equal(got.double()[inf], want[inf]), what
    assert not got[want.isnan()].isfinite().any(), what
    hold(what, torch.where(fine, got, 0), (torch.where(fine, want, 0.0), torch.where(fine, mag, 0.0)))


@pytest.mark.parametrize("t", [5, 40, 300, 2500])
@pytest.mark.parametrize("where", ["h0", "x", "dy", "dh"])
def test_infinite_states_stay_infinite(t, where):
    """Slow channels, and ones whose decay over a span underflows, from a state, a token or a gradient
    that is infinite: inf on and on, as the recurrence has it token by token, and not NaN."""
    d = 70
    dt, g, x, _, h0, _, dy, dh = make(1, t, d, torch.float32)
    lam = torch.linspace(-7, 2.5, d, device=DEV)
    mid = t // 2
    for i, v in enumerate((float("inf"), -float("inf"))):
        {"h0": h0, "x": x[:, mid], "dy": dy[:, mid], "dh": dh}[where][:, i::3] = v
    ref = walk(dt, g, x, lam, h0, None, dy, dh)
    assert ref["y"][0].isnan().sum() == 0
    leaves = [v.requires_grad_() for v in (dt, g, x, lam, h0)]
    y, h = gated_scan(*leaves[:4], h0=h0, return_state=True)
    hold_kinds("y", y.detach(), ref["y"])
    hold_kinds("h", h.detach(), ref["h"])
    for name, got in zip(["dt", "g", "x", "rate", "h0"], torch.autograd.grad([y, h], leaves, [dy, dh])):
        hold_kinds(name, got, ref[name])


@pytest.mark.parametrize("dtype", TYPES)
def test_step_with_infinities(dtype):
    dt, g, x, _, h0, _, _, _ = make(2, 6, 90, dtype)
    lam = torch.linspace(-7, 2.5, 90, device=DEV)
    h0[0, ::3], h0[1, 1::3] = float("inf"), -float("inf")
    x[0, 2, 1::3], x[1, 3, ::3] = float("inf"), -float("inf")
    ref = walk(dt, g, x, lam, h0, None)
    assert ref["y"][0].isnan().sum() == 0
    h = h0.clone()
    for i in range(6):
        y = gated_scan_step_(dt[:, i:i + 1], g[:, i:i + 1], x[:, i:i + 1], lam, h)
        hold_kinds("y", y[:, 0], tuple(v[:, i] for v in ref["y"]))
    hold_kinds("h", h, ref["h"])


def test_forward_mode_is_refused():
    dt, g, x, lam, _, _, dy, _ = make(2, 20, 8, torch.float32)
    y = gated_scan(dt, g, x.requires_grad_(), lam)
    ad = torch.autograd.forward_ad
    with ad.dual_level():
        for grad in (False, True):
            dual = ad.make_dual(x.detach().requires_grad_(grad), torch.ones_like(x))
            with pytest.raises(RuntimeError):
                gated_scan(dt, g, dual, lam)
        with pytest.raises(RuntimeError):  # a gradient with a tangent
            torch.autograd.grad(y, x, ad.make_dual(dy, torch.ones_like(dy)))
    assert gated_scan(dt, g, x, lam).isfinite().all()
