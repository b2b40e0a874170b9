"""The operators of a stack with matrix states, case by case: the gated delta rule (its forward, its
backward, its single-token step), the layer norm with its weights' gradients, and the orthogonalised
update of matrices (alone, and as the optimiser's whole step).

`listed()` names the sizes, `draw(rng)` gives more of the same ranges, `prepare` makes what a program
has in hand, `run` makes one pass (through the framework's entry points where `own` is true, in
elementary torch operations otherwise), `work` says what the pass cannot do without, and `exact` gives
its result from the definition in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
CHUNK = 64  # tokens that the plain form takes together
NORM_EPS = 1e-5
LR, MOMENTUM, DECAY, ORTHO_EPS = 0.02, 0.95, 0.1, 1e-7
STEPS, COEFFICIENTS = 5, (3.4445, -4.7750, 2.0315)


def listed():
    return [
        # A training step's mixer over four full sequences at the base preset's inner width (1536 as
        # twelve heads).
        {"name": "delta_train_bf16", "kind": "delta", "grad": True, "dtype": "bf16", "batch": 4,
         "seq": 2048, "k_heads": 12, "v_heads": 12, "k_dim": 128, "v_dim": 128, "state": False,
         "packed": False},
        # One long prompt, continued from a state and leaving one for the tokens to come; three value
        # heads to a key head.
        {"name": "delta_prompt_bf16", "kind": "delta", "grad": False, "dtype": "bf16", "batch": 1,
         "seq": 16384, "k_heads": 4, "v_heads": 12, "k_dim": 128, "v_dim": 128, "state": True,
         "packed": False},
        # Packed documents of a ragged length and odd widths in fp32, the state carried between steps.
        {"name": "delta_packed_fp32", "kind": "delta", "grad": True, "dtype": "fp32", "batch": 3,
         "seq": 1531, "k_heads": 5, "v_heads": 5, "k_dim": 60, "v_dim": 100, "state": True,
         "packed": True},
        # One token for each of sixteen sequences: the decode loop's latency.
        {"name": "delta_step_fp16", "kind": "step", "dtype": "fp16", "batch": 16, "k_heads": 12,
         "v_heads": 12, "k_dim": 128, "v_dim": 128},
        # The base preset's last norm in training.
        {"name": "norm_train_bf16", "kind": "norm", "grad": True, "dtype": "bf16", "rows": 8192,
         "width": 768, "affine": True},
        # An odd width in fp32, without weight and bias.
        {"name": "norm_odd_fp32", "kind": "norm", "grad": True, "dtype": "fp32", "rows": 3001,
         "width": 515, "affine": False},
        # One token for each of four sequences.
        {"name": "norm_step_fp16", "kind": "norm", "grad": False, "dtype": "fp16", "rows": 4,
         "width": 768, "affine": True},
        # One update of odd shape in fp32, three of them stacked.
        {"name": "ortho_odd_fp32", "kind": "ortho", "dtype": "fp32", "batch": 3, "rows": 515,
         "cols": 1000},
        # Updates of the base preset's inner width, tall, in bf16.
        {"name": "ortho_tall_bf16", "kind": "ortho", "dtype": "bf16", "batch": 12, "rows": 1536,
         "cols": 768},
        # The matrices of one smallest block (width 64) in fp32: launches and latency.
        {"name": "muon_small_fp32", "kind": "muon", "dtype": "fp32", "layers": 1, "d_model": 64},
        # The matrices of the small preset's eight blocks in bf16.
        {"name": "muon_preset_bf16", "kind": "muon", "dtype": "bf16", "layers": 8, "d_model": 512},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["delta", "delta", "step", "norm", "ortho", "muon"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if kind in ("delta", "step"):
        while True:
            c = {"kind": kind, "dtype": dtype, "batch": _log_int(rng, 1, 8 if kind == "delta" else 64),
                 "k_heads": rng.randint(1, 8), "k_dim": _log_int(rng, 16, 128),
                 "v_dim": _log_int(rng, 16, 256)}
            c["v_heads"] = c["k_heads"] * rng.choice([1, 1, 2, 3])
            if kind == "step":
                return c
            c |= {"seq": _log_int(rng, 1, 16384), "grad": rng.random() < 0.6,
                  "state": rng.random() < 0.5, "packed": rng.random() < 0.4}
            lanes = c["batch"] * c["v_heads"] * c["k_dim"] * c["v_dim"]
            if lanes * c["seq"] <= (1 if c["grad"] else 2) * 1536 << 20:
                return c
    if kind == "norm":
        while True:
            rows, width = _log_int(rng, 1, 65536), _log_int(rng, 17, 8192)
            if rows * width <= 16 << 20:
                break
        return {"kind": "norm", "grad": rng.random() < 0.6, "dtype": dtype, "rows": rows,
                "width": width, "affine": rng.random() < 0.8}
    if kind == "ortho":
        while True:
            c = {"kind": "ortho", "dtype": dtype, "batch": rng.randint(1, 16),
                 "rows": _log_int(rng, 17, 2048), "cols": _log_int(rng, 17, 2048)}
            if work(c)["flops"] <= 100e9:
                return c
    return {"kind": "muon", "dtype": dtype, "layers": rng.randint(1, 6),
            "d_model": _log_int(rng, 16, 400)}


# --- what a program has in hand -----------------------------------------------------------------

def _matrices(case):
    """Shapes of a block's projections in the framework (inner width twice d_model): in_proj, the two
    gates, out_proj."""
    d = case["d_model"]
    return [(4 * d, d), (2 * d, 2 * d), (2 * d, 2 * d), (d, 8 * d)]


def _update(gen, shape):
    """What a gradient looks like: some directions far above the others."""
    def rnd(*s):
        return torch.randn(*s, generator=gen, device="cuda")
    *batch, m, n = shape
    few = max(1, min(m, n) // 16)
    size = 10 ** (-1.5 * torch.rand(few, generator=gen, device="cuda"))
    strong = (rnd(*batch, m, few) * size) @ rnd(*batch, few, n)
    return 1e-3 * (rnd(*shape) + 2 * strong)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def rnd32(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def rnd(*shape):
        return rnd32(*shape).to(dtype)

    s = {"case": case}
    if case["kind"] in ("delta", "step"):
        b, t, hk, hv = case["batch"], case.get("seq", 1), case["k_heads"], case["v_heads"]
        dk, dv = case["k_dim"], case["v_dim"]
        # Parts of one projection's output, read in place; queries and keys of length one.
        qkv = rnd32(b, t, 2 * hk * dk + hv * dv)
        qk = qkv[..., :2 * hk * dk].unflatten(-1, (2 * hk, dk))
        qk /= qk.norm(dim=-1, keepdim=True)
        qkv = qkv.to(dtype)
        qk, s["v"] = qkv[..., :2 * hk * dk], qkv[..., 2 * hk * dk:].unflatten(-1, (hv, dv))
        s["q"], s["k"] = qk.unflatten(-1, (2, hk, dk)).unbind(2)
        # Heads that forget within some tokens and ones that hold for thousands.
        rate = 10 ** (-3.5 * torch.rand(hv, generator=gen, device="cuda"))
        s["log_decay"] = -rate * (rnd32(b, t, hv) - 1).exp()
        s["beta"] = torch.sigmoid(rnd32(b, t, hv)).to(dtype)
        s["h0"] = 0.3 * rnd32(b, hv, dk, dv) if case["kind"] == "step" or case["state"] else None
        if case["kind"] == "step":
            return s
        s["reset"] = (torch.rand(b, t, generator=gen, device="cuda") < 1 / 300
                      if case["packed"] else None)
        if case["grad"]:
            s["do"] = rnd(b, t, hv, dv)
            s["dh"] = rnd32(b, hv, dk, dv) if case["state"] else None
            for k in ("q", "k", "v", "log_decay", "beta", "h0"):
                s[k] = None if s[k] is None else s[k].detach().requires_grad_()
        return s
    if case["kind"] == "norm":
        n, d = case["rows"], case["width"]
        s["x"] = (rnd32(n, d) * 2 + rnd32(n, 1)).to(dtype)
        s["weight"] = 1 + 0.2 * rnd32(d) if case["affine"] else None
        s["bias"] = 0.2 * rnd32(d) if case["affine"] else None
        if case["grad"]:
            s["dy"] = rnd(n, d)
            for k in ("x", "weight", "bias"):
                s[k] = None if s[k] is None else s[k].requires_grad_()
        return s
    if case["kind"] == "ortho":
        s["x"] = _update(gen, (case["batch"], case["rows"], case["cols"])).to(dtype)
        return s
    for k in ("p", "grad", "m"):
        s[k] = []
    for shape in _matrices(case):
        shape = (case["layers"], *shape)
        s["p"].append((0.02 * rnd32(*shape)).to(dtype))
        grad = _update(gen, shape)
        s["grad"].append(grad.to(dtype))
        s["m"].append(0.5 * grad + 0.5 * _update(gen, shape))
    for k in ("p", "grad", "m"):
        s[k + "s"] = [x for stack in s[k] for x in stack.unbind()]
    return s


# --- one pass -----------------------------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"delta": _delta_own, "step": _step_own, "norm": _norm_own, "ortho": _ortho_own,
                "muon": _muon_own}[kind](s)
    if kind == "delta":
        with torch.set_grad_enabled(s["case"]["grad"]):
            return _delta_plain(s)
    with torch.no_grad():
        return {"step": _step_plain, "norm": _norm_plain, "ortho": _ortho_plain,
                "muon": _muon_plain}[kind](s)


def _delta_own(s):
    from mambaqc_amd.kernels import gated_delta
    c = s["case"]
    with torch.set_grad_enabled(c["grad"]):
        o, h = gated_delta(s["q"], s["k"], s["v"], s["log_decay"], s["beta"], h0=s["h0"],
                           reset=s["reset"], return_state=True)
    return _with_grads(s, o, h)


def _with_grads(s, o, h):
    c = s["case"]
    if not c["grad"]:
        return {"o": o, "h": h}
    names = ["q", "k", "v", "log_decay", "beta"] + (["h0"] if c["state"] else [])
    ends, grads = ([o, h], [s["do"], s["dh"]]) if c["state"] else ([o], [s["do"]])
    got = torch.autograd.grad(ends, [s[k] for k in names], grads)
    return {"o": o.detach(), "h": h.detach(), **{"d" + k: v for k, v in zip(names, got)}}


def _step_own(s):
    from mambaqc_amd.kernels import gated_delta_step_
    o = gated_delta_step_(s["q"], s["k"], s["v"], s["log_decay"], s["beta"], s["h0"])
    return {"o": o, "h": s["h0"]}


def _norm_own(s):
    from mambaqc_amd.kernels import layer_norm
    if not s["case"]["grad"]:
        with torch.no_grad():
            return {"y": layer_norm(s["x"], s["weight"], s["bias"], eps=NORM_EPS)}
    y = layer_norm(s["x"], s["weight"], s["bias"], eps=NORM_EPS)
    names = [k for k in ("x", "weight", "bias") if s[k] is not None]
    got = torch.autograd.grad(y, [s[k] for k in names], s["dy"])
    return {"y": y.detach(), **{"d" + k: v for k, v in zip(names, got)}}


def _ortho_own(s):
    from mambaqc_amd.optim import orthogonalize
    return {"x": orthogonalize(s["x"], steps=STEPS, coefficients=COEFFICIENTS, eps=ORTHO_EPS)}


def _muon_own(s):
    from mambaqc_amd.optim import muon_step_
    muon_step_(s["ps"], s["grads"], s["ms"], lr=LR, momentum=MOMENTUM, nesterov=True,
               weight_decay=DECAY, steps=STEPS, coefficients=COEFFICIENTS, eps=ORTHO_EPS)
    return {"p": s["p"], "m": s["m"]}


def _chunked(x, length):
    """[b, t, h, ..] as [b, h, chunks, CHUNK, ..], the end filled with zeros."""
    x = x.transpose(1, 2)
    if length > x.shape[2]:
        x = torch.cat([x, x.new_zeros(*x.shape[:2], length - x.shape[2], *x.shape[3:])], 2)
    return x.unflatten(2, (-1, CHUNK))


def _delta_plain(s):
    """Chunks of 64 tokens: within one, what the tokens write from a triangular system; from one to the
    next, the state goes through an affine map, and these are joined by doubling."""
    c = s["case"]
    t, group = c["seq"], c["v_heads"] // c["k_heads"]
    length = -(-t // CHUNK) * CHUNK
    q, k = (_chunked(s[n].float().repeat_interleave(group, 2), length) for n in ("q", "k"))
    v, beta = _chunked(s["v"].float(), length), _chunked(s["beta"].float(), length)[..., None]
    total = _chunked(s["log_decay"].double(), length).cumsum(-1)
    if s["reset"] is None:
        doc = torch.zeros(1, 1, length // CHUNK, CHUNK, dtype=torch.int32, device="cuda")
    else:
        doc = _chunked(s["reset"].int()[..., None], length).cumsum(-1)
    at = torch.arange(CHUNK, device="cuda")
    seen = (doc[..., :, None] == doc[..., None, :]) & (at[:, None] >= at)
    decay = torch.where(seen, total[..., :, None] - total[..., None, :], -math.inf).exp().float()
    into = torch.where(doc == 0, total, -math.inf).exp().float()[..., None]
    last, all_of_it = decay[..., -1, :, None], into[..., -1:, :]
    kt = k.transpose(-1, -2)
    system = -beta * decay * (k @ kt) * (at[:, None] > at)
    inverse = torch.eye(CHUNK, device="cuda") + system
    for _ in range(5):
        system = system @ system
        inverse = inverse + inverse @ system
    w, u = inverse @ (beta * into * k), inverse @ (beta * v)
    back = (last * k).transpose(-1, -2)
    m = all_of_it * torch.eye(c["k_dim"], device="cuda") - back @ w
    n = back @ u
    first = (torch.zeros_like(n[:, :, :1]) if s["h0"] is None else s["h0"][:, :, None])
    n = torch.cat([first, n], 2)
    m = torch.cat([torch.zeros_like(m[:, :, :1]), m], 2)
    step = 1
    while step < n.shape[2]:
        n = torch.cat([n[:, :, :step], n[:, :, step:] + m[:, :, step:] @ n[:, :, :-step]], 2)
        m = torch.cat([m[:, :, :step], m[:, :, step:] @ m[:, :, :-step]], 2)
        step *= 2
    h, start = n[:, :, -1], n[:, :, :-1]
    o = into * (q @ start) + (decay * (q @ kt)) @ (u - w @ start)
    o = (o * c["k_dim"] ** -0.5).flatten(2, 3)[:, :, :t].transpose(1, 2)
    return _with_grads(s, o.to(s["v"].dtype).contiguous(), h)


def _step_plain(s):
    c, h = s["case"], s["h0"]
    group = c["v_heads"] // c["k_heads"]
    q, k = (s[n].float().repeat_interleave(group, 2)[:, 0, :, :, None] for n in ("q", "k"))
    v, beta = s["v"].float()[:, 0, :, None], s["beta"].float()[:, 0, :, None, None]
    h.mul_(s["log_decay"].exp()[:, 0, :, None, None])
    h.add_(k * (beta * (v - (h * k).sum(2, keepdim=True))))
    o = (h * q).sum(2)[:, None] * c["k_dim"] ** -0.5
    return {"o": o.to(s["v"].dtype), "h": h}


def _norm_plain(s):
    x = s["x"].float()
    x = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((x * x).mean(1, keepdim=True) + NORM_EPS)
    hat = x * rstd
    y = hat if s["weight"] is None else hat * s["weight"] + s["bias"]
    out = {"y": y.to(s["x"].dtype)}
    if not s["case"]["grad"]:
        return out
    dy = s["dy"].float()
    g = dy if s["weight"] is None else dy * s["weight"]
    dx = rstd * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
    out["dx"] = dx.to(s["x"].dtype)
    if s["weight"] is not None:
        out |= {"dweight": (dy * hat).sum(0), "dbias": dy.sum(0)}
    return out


def _ortho(x):
    """Newton and Schulz's iteration towards the nearest orthogonal matrix, in x's type."""
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2).contiguous() if tall else x
    x = x / (x * x).sum((-2, -1), keepdim=True).sqrt().clamp_min(ORTHO_EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        gram = x @ x.transpose(-1, -2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-1, -2).contiguous() if tall else x


def _ortho_plain(s):
    return {"x": _ortho(s["x"].float()).to(s["x"].dtype)}


def _muon_plain(s):
    for p, grad, m in zip(s["p"], s["grad"], s["m"]):
        g = grad.float()
        m.mul_(MOMENTUM).add_(g * (1 - MOMENTUM))
        x = _ortho(m * MOMENTUM + g * (1 - MOMENTUM))
        size = max(1, p.shape[-2] / p.shape[-1]) ** 0.5
        p.copy_(p.float() * (1 - LR * DECAY) - x * (LR * size))
    return {"p": s["p"], "m": s["m"]}


# --- the work of a pass, and its result in 64 bits ----------------------------------------------

def _ortho_flops(m, n):
    """Of the products' two symmetric results half is enough."""
    m, n = min(m, n), max(m, n)
    return STEPS * (3 * m * m * n + m * m * m)


def work(case):
    e = BYTES[case["dtype"]]
    if case["kind"] in ("delta", "step"):
        b, t, hk, hv = case["batch"], case.get("seq", 1), case["k_heads"], case["v_heads"]
        dk, dv = case["k_dim"], case["v_dim"]
        grad, lanes = case.get("grad", False), b * hv * dk * dv
        states = 2 if case["kind"] == "step" or case["state"] else 1
        total = b * t * (2 * hk * dk * e + 2 * hv * dv * e + hv * (4 + e)) + lanes * 4 * states
        if grad:
            total += b * t * (2 * hk * dk * e + 2 * hv * dv * e + hv * (4 + e))
            total += lanes * 8 * case["state"]
        if case.get("packed"):
            total += b * t
        # A token's products with the state: two that write it, one that reads it.
        flops = b * t * hv * dk * dv * 6
        return {"bytes": total, "flops": flops * (3 if grad else 1)}
    if case["kind"] == "norm":
        n, d = case["rows"] * case["width"], case["width"]
        weights = 2 * case["affine"] * (2 if case["grad"] else 1)
        return {"bytes": n * e * (4 if case["grad"] else 2) + d * 4 * weights,
                "flops": n * (20 if case["grad"] else 8)}
    if case["kind"] == "ortho":
        n = case["batch"] * case["rows"] * case["cols"]
        return {"bytes": 2 * n * e, "flops": case["batch"] * _ortho_flops(case["rows"], case["cols"])}
    shapes = _matrices(case)
    n = case["layers"] * sum(x * y for x, y in shapes)
    return {"bytes": n * (3 * e + 8),
            "flops": case["layers"] * sum(_ortho_flops(x, y) for x, y in shapes)}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] in ("delta", "step"):
            return _delta_exact(s)
        if case["kind"] == "norm":
            return _norm_exact(s)
        if case["kind"] == "ortho":
            return {"x": _ortho_exact(s["x"])}
        return _muon_exact(s)


def _delta_exact(s):
    """The recurrence token by token, and its adjoint."""
    c = s["case"]
    group = c["v_heads"] // c["k_heads"]
    q, k, v, g, beta = (s[n].detach().double() for n in ("q", "k", "v", "log_decay", "beta"))
    q = torch.repeat_interleave(q, group, 2) * c["k_dim"] ** -0.5
    k = torch.repeat_interleave(k, group, 2)
    b, t, h, dv = v.shape
    a = g.exp()
    if s.get("reset") is not None:
        a = torch.where(s["reset"][..., None], 0.0, a)
    state = (v.new_zeros(b, h, c["k_dim"], dv) if s["h0"] is None else s["h0"].detach().double())
    o, states = torch.empty_like(v), []
    for i in range(t):
        if c.get("grad"):
            states.append(state)
        state = state * a[:, i, :, None, None]
        r = v[:, i] - torch.matmul(k[:, i, :, None], state)[:, :, 0]
        state = torch.addcmul(state, k[:, i, :, :, None], (beta[:, i, :, None] * r)[:, :, None])
        o[:, i] = torch.matmul(q[:, i, :, None], state)[:, :, 0]
    out = {"o": o, "h": state}
    if not c.get("grad"):
        return out
    bar = v.new_zeros(state.shape) if s["dh"] is None else s["dh"].double()
    do = s["do"].double()
    dq, dk, dv_, da, dbeta = (torch.empty_like(x) for x in (q, k, v, a, beta))
    for i in reversed(range(t)):
        before, ki, wi = states[i], k[:, i, :, :, None], beta[:, i, :, None, None]
        part = before * a[:, i, :, None, None]
        r = v[:, i, :, None] - (part * ki).sum(2, keepdim=True)
        after = part + ki * wi * r
        dq[:, i] = (after * do[:, i, :, None]).sum(-1)
        bar = bar + q[:, i, :, :, None] * do[:, i, :, None]
        dw = (bar * ki).sum(2, keepdim=True)
        dbeta[:, i] = (dw * r).sum((-2, -1))
        dr = wi * dw
        dv_[:, i] = dr[:, :, 0]
        dk[:, i] = (bar * wi * r - part * dr).sum(-1)
        bar = bar - ki * dr
        da[:, i] = (bar * before).sum((-2, -1))
        bar = bar * a[:, i, :, None, None]
    shared = (lambda x: x.unflatten(2, (-1, group)).sum(3))
    out |= {"dq": shared(dq) * c["k_dim"] ** -0.5, "dk": shared(dk), "dv": dv_,
            "dlog_decay": da * a, "dbeta": dbeta}
    if s["h0"] is not None:
        out["dh0"] = bar
    return out


def _norm_exact(s):
    """Values from the definition, gradients by differentiating it."""
    grad = s["case"]["grad"]
    leaves = {k: s[k].detach().double().requires_grad_(grad)
              for k in ("x", "weight", "bias") if s[k] is not None}
    with torch.set_grad_enabled(grad):
        x = leaves["x"]
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        y = (x - mean) / (var + NORM_EPS).sqrt()
        if "weight" in leaves:
            y = torch.addcmul(leaves["bias"], y, leaves["weight"])
        got = {"y": y.detach()}
        if grad:
            grads = torch.autograd.grad(y, list(leaves.values()), s["dy"].double())
            got |= {"d" + k: v for k, v in zip(leaves, grads)}
    return got


def _ortho_exact(x):
    """The iteration from the side of the smaller Gram matrix, no transposes taken of x itself."""
    x = x.double()
    x = x / torch.linalg.matrix_norm(x, keepdim=True).clamp_min(ORTHO_EPS)
    for _ in range(STEPS):
        if x.shape[-2] > x.shape[-1]:
            gram = torch.matmul(x.mT.contiguous(), x)
            right = COEFFICIENTS[1] * gram + COEFFICIENTS[2] * torch.matmul(gram, gram)
            x = COEFFICIENTS[0] * x + torch.matmul(x, right)
        else:
            gram = torch.matmul(x, x.mT.contiguous())
            left = COEFFICIENTS[1] * gram + COEFFICIENTS[2] * torch.matmul(gram, gram)
            x = COEFFICIENTS[0] * x + torch.matmul(left, x)
    return x


def _muon_exact(s):
    out = {"p": [], "m": []}
    for p, grad, m in zip(s["p"], s["grad"], s["m"]):
        g = grad.double()
        m = torch.lerp(g, m.double(), MOMENTUM)
        x = _ortho_exact(torch.lerp(g, m, MOMENTUM))
        rows, cols = p.shape[-2:]
        out["m"].append(m)
        out["p"].append((1 - LR * DECAY) * p.double() - LR * math.sqrt(max(1, rows / cols)) * x)
    return out
