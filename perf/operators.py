"""The operators of a recurrent stack's training and serving, case by case: the gated scan (its
forward, its backward, its single-token step), the gate, norms and residual between two blocks, and
the AdamW step with states in 32 or in 8 bits.

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
NORM_EPS = 1e-6
LR, BETA1, BETA2, ADAM_EPS, DECAY, MAX_NORM = 3e-4, 0.9, 0.95, 1e-8, 0.1, 1.0
BLOCK = 256  # elements that share a scale in the 8-bit states


def listed():
    return [
        # A training step's scan over four full sequences at the base preset's inner width.
        {"name": "scan_train_bf16", "kind": "scan", "grad": True, "dtype": "bf16", "batch": 4,
         "seq": 2048, "width": 1536, "state": False, "packed": False},
        # One long prompt, continued from a state and leaving one for the tokens to come.
        {"name": "scan_prompt_bf16", "kind": "scan", "grad": False, "dtype": "bf16", "batch": 1,
         "seq": 16384, "width": 1536, "state": True, "packed": False},
        # Packed documents of a ragged length in fp32, the state carried between steps.
        {"name": "scan_packed_fp32", "kind": "scan", "grad": True, "dtype": "fp32", "batch": 3,
         "seq": 1531, "width": 500, "state": True, "packed": True},
        # One token for each of sixteen sequences: the decode loop's latency.
        {"name": "scan_step_fp16", "kind": "step", "dtype": "fp16", "batch": 16, "width": 1536},
        # Between two blocks of the base preset in training.
        {"name": "norm_train_bf16", "kind": "norm", "grad": True, "dtype": "bf16", "rows": 8192,
         "width": 768, "gate": True, "post": True},
        # The same in a prompt's forward pass, many rows of the large preset's width.
        {"name": "norm_prompt_fp16", "kind": "norm", "grad": False, "dtype": "fp16",
         "rows": 32768, "width": 1024, "gate": True, "post": True},
        # An odd width in fp32, without a gate.
        {"name": "norm_odd_fp32", "kind": "norm", "grad": True, "dtype": "fp32", "rows": 3001,
         "width": 515, "gate": False, "post": True},
        # One token for each of four sequences.
        {"name": "norm_step_bf16", "kind": "norm", "grad": False, "dtype": "bf16", "rows": 4,
         "width": 768, "gate": True, "post": True},
        # The parameters of one smallest block (width 64, 16 states), in fp32: launches and latency.
        {"name": "adamw_small_fp32", "kind": "adamw", "dtype": "fp32", "bits": 32, "clip": False,
         "layers": 1, "d_model": 64, "d_state": 16, "vocab": 0},
        # A small model in fp32 with its gradients' norm clipped.
        {"name": "adamw_model_fp32", "kind": "adamw", "dtype": "fp32", "bits": 32, "clip": True,
         "layers": 4, "d_model": 128, "d_state": 16, "vocab": 10000},
        # The same kind of model with 8-bit states.
        {"name": "adamw8_model_fp32", "kind": "adamw", "dtype": "fp32", "bits": 8, "clip": True,
         "layers": 3, "d_model": 96, "d_state": 16, "vocab": 4999},
        # One block of the small preset in bf16 with 8-bit states: 273 million parameters.
        {"name": "adamw8_block_bf16", "kind": "adamw", "dtype": "bf16", "bits": 8, "clip": False,
         "layers": 1, "d_model": 512, "d_state": 32, "vocab": 0},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["scan", "scan", "norm", "adamw"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if kind == "scan":
        if rng.random() < 0.2:
            return {"kind": "step", "dtype": dtype, "batch": _log_int(rng, 1, 64),
                    "width": _log_int(rng, 17, 4096)}
        while True:
            batch, seq = rng.randint(1, 8), _log_int(rng, 1, 16384)
            width = _log_int(rng, 17, 4096)
            if batch * seq * width <= 12 << 20:
                break
        return {"kind": "scan", "grad": rng.random() < 0.6, "dtype": dtype, "batch": batch,
                "seq": seq, "width": width, "state": rng.random() < 0.5,
                "packed": rng.random() < 0.4}
    if kind == "norm":
        while True:
            rows, width = _log_int(rng, 1, 65536), _log_int(rng, 17, 8192)
            if rows * width <= 16 << 20:
                break
        return {"kind": "norm", "grad": rng.random() < 0.6, "dtype": dtype, "rows": rows,
                "width": width, "gate": rng.random() < 0.7, "post": rng.random() < 0.8}
    while True:
        case = {"kind": "adamw", "dtype": dtype, "bits": rng.choice([8, 32]),
                "clip": rng.random() < 0.5, "layers": rng.randint(1, 6),
                "d_model": _log_int(rng, 16, 320), "d_state": _log_int(rng, 4, 32),
                "vocab": rng.choice([0, _log_int(rng, 101, 20011)])}
        if sum(_sizes(case)) <= 60 << 20:
            return case


# --- what a program has in hand -----------------------------------------------------------------

def _sizes(case):
    """Elements of each parameter of `layers` blocks of the framework (inner width twice d_model),
    and of an embedding."""
    d, n, di = case["d_model"], case["d_state"], 2 * case["d_model"]
    block = [2 * di * d, 4 * di, di, di * di, di * di, di * n * 4 * di, di * n * 4 * di, di * n,
             di * n * 3, di, di, 4 * di, d * 4 * di]
    return block * case["layers"] + ([case["vocab"] * d] if case["vocab"] else [])


def _random(gen, dtype):
    return lambda *shape: torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES.get(case["dtype"])
    rnd, rnd32 = _random(gen, dtype), _random(gen, torch.float32)
    s = {"case": case}
    if case["kind"] in ("scan", "step"):
        b, t, d = case["batch"], case.get("seq", 1), case["width"]
        s["dt"] = (rnd32(b, t, d) * 1.5 - 1).to(dtype)
        s["g"], s["x"] = rnd(b, t, d), rnd(b, t, d)
        # Rates over three decades: channels that forget within a token and ones that hold for
        # thousands.
        s["log_rate"] = torch.rand(d, generator=gen, device="cuda") * math.log(2e3) + math.log(1e-3)
        s["h0"] = rnd32(b, d) if case["kind"] == "step" or case["state"] else None
        if case["kind"] == "step":
            return s
        s["reset"] = (torch.rand(b, t, generator=gen, device="cuda") < 1 / 300
                      if case["packed"] else None)
        if case["grad"]:
            s["dy"], s["dh"] = rnd(b, t, d), rnd32(b, d) if case["state"] else None
            for k in ("dt", "g", "x", "log_rate", "h0"):
                s[k] = None if s[k] is None else s[k].requires_grad_()
        return s
    if case["kind"] == "norm":
        n, d = case["rows"], case["width"]
        s["x"], s["y"] = rnd(n, d), rnd(n, d)
        # The gate is the second half of a projection's output, read in place.
        s["z"] = rnd(n, 2 * d)[:, d:] if case["gate"] else None
        s["post"] = 1 + 0.2 * rnd32(d) if case["post"] else None
        s["scale"], s["pre"] = 0.3 + 0.1 * rnd32(d), 1 + 0.2 * rnd32(d)
        if case["grad"]:
            s["dout"], s["dn"] = rnd(n, d), rnd(n, d)
            for k in ("x", "y", "z", "post", "scale", "pre"):
                s[k] = None if s[k] is None else s[k].requires_grad_()
        return s
    # The tensors of a model as views of flat buffers, each starting at a multiple of BLOCK.
    sizes = _sizes(case)
    starts, total = [], 0
    for k in sizes:
        starts.append(total)
        total += -(-k // BLOCK) * BLOCK
    s["sizes"], s["starts"] = sizes, starts
    s["step"] = 100 + seed % 1000
    used = torch.zeros(total, dtype=torch.bool, device="cuda")
    s["p"] = torch.zeros(total, dtype=dtype, device="cuda")
    s["grad"] = torch.zeros(total, dtype=dtype, device="cuda")
    m = torch.zeros(total, device="cuda")
    v = torch.zeros(total, device="cuda")
    for at, k in zip(starts, sizes):
        used[at:at + k] = True
        size = 10 ** (-4 + 2 * torch.rand(1, generator=gen, device="cuda"))
        s["p"][at:at + k] = (0.02 * rnd32(k)).to(dtype)
        s["grad"][at:at + k] = (size * rnd32(k)).to(dtype)
        m[at:at + k] = 0.3 * size * rnd32(k)
        v[at:at + k] = (size * (1 + 0.3 * rnd32(k))) ** 2
    del used
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        for name, value in (("m", m), ("v", v.sqrt())):
            top = value.view(-1, BLOCK).abs().amax(1).clamp_min(2.0 ** -100)
            scale = torch.exp2(torch.ceil(torch.log2(top / 448)))
            s[name] = (value.view(-1, BLOCK) / scale[:, None]).to(torch.float8_e4m3fn).view(-1)
            s[name + "_scale"] = scale
    for k in ("p", "grad", "m", "v"):
        s[k + "s"] = [s[k][at:at + n] for at, n in zip(starts, sizes)]
    if case["bits"] == 8:
        for k in ("m_scale", "v_scale"):
            s[k + "s"] = [s[k][at // BLOCK:at // BLOCK + -(-n // BLOCK)]
                          for at, n in zip(starts, sizes)]
        # Which element of its tensor each element of the flat buffers is, for the rounding.
        s["seed"] = seed
        lengths = torch.tensor([-(-k // BLOCK) * BLOCK for k in sizes], device="cuda")
        s["first"] = torch.repeat_interleave(torch.tensor(starts, device="cuda"), lengths // BLOCK)
        s["which"] = torch.repeat_interleave(torch.arange(len(sizes), device="cuda"),
                                             lengths // BLOCK)
    return s


# --- one pass -----------------------------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if own:
        if kind == "step":
            return _step_own(s)
        if kind == "scan":
            return _scan_own(s)
        return _norm_own(s) if kind == "norm" else _adamw_own(s)
    with torch.no_grad():
        if kind in ("scan", "step"):
            return _scan_plain(s)
        return _norm_plain(s) if kind == "norm" else _adamw_plain(s)


def _step_own(s):
    from mambaqc_amd.kernels import gated_scan_step_
    y = gated_scan_step_(s["dt"], s["g"], s["x"], s["log_rate"], s["h0"])
    return {"y": y, "h": s["h0"]}


def _scan_own(s):
    from mambaqc_amd.kernels import gated_scan
    c = s["case"]
    if not c["grad"]:
        with torch.no_grad():
            y, h = gated_scan(s["dt"], s["g"], s["x"], s["log_rate"], h0=s["h0"],
                              reset=s["reset"], return_state=True)
        return {"y": y, "h": h}
    y, h = gated_scan(s["dt"], s["g"], s["x"], s["log_rate"], h0=s["h0"], reset=s["reset"],
                      return_state=True)
    names = ["dt", "g", "x", "log_rate"] + (["h0"] if c["state"] else [])
    ends, grads = ([y, h], [s["dy"], s["dh"]]) if c["state"] else ([y], [s["dy"]])
    got = torch.autograd.grad(ends, [s[k] for k in names], grads)
    return {"y": y, "h": h, **{"d" + k: v for k, v in zip(names, got)}}


def _norm_own(s):
    from mambaqc_amd.kernels import gate_norm_residual
    if not s["case"]["grad"]:
        with torch.no_grad():
            out, n = gate_norm_residual(s["x"], s["y"], s["z"], post_weight=s["post"],
                                        scale=s["scale"], pre_weight=s["pre"], eps=NORM_EPS)
        return {"out": out, "n": n}
    out, n = gate_norm_residual(s["x"], s["y"], s["z"], post_weight=s["post"], scale=s["scale"],
                                pre_weight=s["pre"], eps=NORM_EPS)
    names = [k for k in ("x", "y", "z", "post", "scale", "pre") if s[k] is not None]
    got = torch.autograd.grad([out, n], [s[k] for k in names], [s["dout"], s["dn"]])
    return {"out": out, "n": n, **{"d" + k: v for k, v in zip(names, got)}}


def _adamw_own(s):
    from mambaqc_amd.optim import adamw8_step_, adamw_step_
    c = s["case"]
    s["step"] += 1
    how = {"step": s["step"], "lr": LR, "betas": (BETA1, BETA2), "eps": ADAM_EPS,
           "weight_decay": DECAY, "max_norm": MAX_NORM if c["clip"] else None}
    if c["bits"] == 32:
        norm = adamw_step_(s["ps"], s["grads"], s["ms"], s["vs"], **how)
        return {"p": s["p"], "m": s["m"], "v": s["v"], "norm": norm}
    norm = adamw8_step_(s["ps"], s["grads"], s["ms"], s["m_scales"], s["vs"], s["v_scales"],
                        seed=s["seed"], **how)
    return {"p": s["p"], "m": s["m"], "m_scale": s["m_scale"], "v": s["v"],
            "v_scale": s["v_scale"], "norm": norm}


def _walk(a, u):
    """h_t = a_t h_{t-1} + u_t along axis 1, from zero, by doubling."""
    n = 1
    while n < u.shape[1]:
        u = torch.cat([u[:, :n], torch.addcmul(u[:, n:], a[:, n:], u[:, :-n])], 1)
        a = torch.cat([a[:, :n], a[:, n:] * a[:, :-n]], 1)
        n *= 2
    return u


def _scan_plain(s):
    c = s["case"]
    dt, g, x = s["dt"].float(), s["g"].float(), s["x"].float()
    rate, h0, reset = torch.exp(s["log_rate"]), s["h0"], s.get("reset")
    p = (dt.clamp_min(0) + torch.log1p(torch.exp(-dt.abs()))) * rate
    a, w = torch.exp(-p), -torch.expm1(-p)
    gate = 1 / (1 + torch.exp(-g))
    sel = gate * x
    keep = a if reset is None else a * ~reset[..., None]
    if c["kind"] == "step":
        s["h0"].copy_((a * h0[:, None] + w * sel)[:, 0])
        return {"y": s["h0"][:, None].to(s["x"].dtype), "h": s["h0"]}
    u = w * sel
    if h0 is not None:
        u[:, 0] += keep[:, 0] * h0
    h = _walk(keep, u)
    out = {"y": h.to(s["x"].dtype), "h": h[:, -1].clone()}
    if not c["grad"]:
        return out
    adj = s["dy"].float()
    if s["dh"] is not None:
        adj = torch.cat([adj[:, :-1], (adj[:, -1] + s["dh"])[:, None]], 1)
    later = torch.cat([keep[:, 1:], torch.zeros_like(keep[:, :1])], 1)
    adj = _walk(later.flip(1), adj.flip(1)).flip(1)
    prev = torch.cat([torch.zeros_like(h[:, :1]) if h0 is None else h0[:, None], h[:, :-1]], 1)
    if reset is not None:
        prev = prev * ~reset[..., None]
    dp = adj * a * (sel - prev)
    dsel = adj * w
    out |= {"ddt": (dp * rate / (1 + torch.exp(-dt))).to(dt_of(s)),
            "dg": (dsel * sel * (1 - gate)).to(dt_of(s)), "dx": (dsel * gate).to(dt_of(s)),
            "dlog_rate": (dp * p).sum((0, 1))}
    if h0 is not None:
        out["dh0"] = keep[:, 0] * adj[:, 0]
    return out


def dt_of(s):
    return DTYPES[s["case"]["dtype"]]


def _norm_plain(s):
    c = s["case"]
    x, y = s["x"].float(), s["y"].float()
    gate = 1 / (1 + torch.exp(-s["z"].float())) if c["gate"] else 1.0
    v = gate * y
    rho = torch.rsqrt((v * v).mean(1, keepdim=True) + NORM_EPS) if c["post"] else 1.0
    r = v * rho * s["post"] if c["post"] else v
    o = x + s["scale"] * r
    tau = torch.rsqrt((o * o).mean(1, keepdim=True) + NORM_EPS)
    out = {"out": o.to(dt_of(s)), "n": (o * tau * s["pre"]).to(dt_of(s))}
    if not c["grad"]:
        return out
    dn = s["dn"].float()
    hat = dn * s["pre"]
    do = s["dout"].float() + tau * hat - o * tau ** 3 * (hat * o).mean(1, keepdim=True)
    dr = s["scale"] * do
    if c["post"]:
        hat = dr * s["post"]
        dv = rho * hat - v * rho ** 3 * (hat * v).mean(1, keepdim=True)
        out["dpost"] = (dr * v * rho).sum(0)
    else:
        dv = dr
    out |= {"dx": do.to(dt_of(s)), "dy": (dv * gate).to(dt_of(s)), "dscale": (do * r).sum(0),
            "dpre": (dn * o * tau).sum(0)}
    if c["gate"]:
        out["dz"] = (dv * v * (1 - gate)).to(dt_of(s))
    return out


def _adamw_plain(s):
    c = s["case"]
    s["step"] += 1
    f = [1 - LR * DECAY, LR / (1 - BETA1 ** s["step"]), 1 / math.sqrt(1 - BETA2 ** s["step"])]
    p, g, norm = s["p"].float(), s["grad"].float(), None
    if c["clip"]:
        # The norm in 64 bits: what is clipped by it lands next to rounding borders.
        total = g.double().square().sum().sqrt()
        norm = total.float()
        g = g * (MAX_NORM / (total + 1e-6)).clamp_max(1).float()
    if c["bits"] == 32:
        m = s["m"].mul_(BETA1).add_(g * (1 - BETA1))
        v = s["v"].mul_(BETA2).add_(g * g * (1 - BETA2))
        root = v.sqrt()
    else:
        m = (s["m"].float().view(-1, BLOCK) * s["m_scale"][:, None]).view(-1)
        root = (s["v"].float().view(-1, BLOCK) * s["v_scale"][:, None]).view(-1)
        m = m * BETA1 + g * (1 - BETA1)
        root = (root * root * BETA2 + g * g * (1 - BETA2)).sqrt()
    s["p"].copy_(p * f[0] - m / (root * f[2] + ADAM_EPS) * f[1])
    if c["bits"] == 32:
        return {"p": s["p"], "m": m, "v": v, "norm": norm}
    _encode(s, m, root)
    return {"p": s["p"], "m": s["m"], "m_scale": s["m_scale"], "v": s["v"],
            "v_scale": s["v_scale"], "norm": norm}


def _power(bits):
    """The floats whose exponent fields are `bits`."""
    return (bits << 23).to(torch.int32).view(torch.float32)


def _field(x):
    return x.view(torch.int32).long() >> 23 & 255


def _scaled(x):
    """|x| under its block's power of two, at most 448 there, and the powers."""
    x = x.view(-1, BLOCK).abs()
    top = x.amax(1)
    bits = (_field(top) + ((top.view(torch.int32) & 0x7fffff) > 0x600000) - 8).clamp_min(1)
    return x * _power(254 - bits)[:, None], _power(bits)


def _steps(x):
    """x in steps of an e4m3 number of its size, and what the binade adds to the code."""
    field = _field(x).clamp_min(121)
    return x * _power(257 - field), (field - 121) << 3


def _encode(s, m, root):
    """The states' new codes. Each value goes to one of the two codes about it, by a number that is
    made from the element's place, the seed and the step: m so that its mean is kept, sqrt(v) so
    that v's is, and never to zero."""
    low, n = 0xffffffff, s["m"].numel()
    at = torch.arange(n, device="cuda").view(-1, BLOCK) - s["first"][:, None]
    r = ((at & low) + ((s["seed"] + s["which"]) * 0x9e3779b9 & low)[:, None]
         + (at >> 32) * 0xbb67ae85) & low
    r = (r ^ r >> 16) * 0x6a09e667 & low
    r = (r ^ r >> 15) * 0xbb67ae85 & low
    r = r ^ r >> 16
    um = ((r + s["step"] * 0x9e3779b9 & low) >> 8).float() * 2.0 ** -24
    r = (r << 16 & low) | r >> 16
    uv = ((r + s["step"] * 0xbb67ae85 & low) >> 8).float() * 2.0 ** -24
    x, scale = _scaled(m)
    s["m_scale"].copy_(scale)
    q, base = _steps(x)
    code = base + (q + um).floor().long() | (m.view(-1, BLOCK) < 0).long() << 7
    s["m"].copy_(code.to(torch.uint8).view(torch.float8_e4m3fn).view(-1))
    x, scale = _scaled(root)
    s["v_scale"].copy_(scale)
    q, base = _steps(x)
    k = q.floor()
    k = k + (uv * (2 * k + 1) < (q - k) * (q + k))
    code = (base + k.long()).clamp_min(1) * (x > 0)
    s["v"].copy_(code.to(torch.uint8).view(torch.float8_e4m3fn).view(-1))


# --- the work of a pass, and its result in 64 bits ----------------------------------------------

def work(case):
    e = BYTES[case["dtype"]]
    if case["kind"] in ("scan", "step"):
        n, lanes = case["batch"] * case.get("seq", 1) * case["width"], case["batch"] * case["width"]
        grad = case.get("grad", False)
        states = 2 if case["kind"] == "step" or case["state"] else 1
        total = n * e * (8 if grad else 4) + case["width"] * 4 + lanes * 4 * states
        if grad:
            total += case["width"] * 4 + lanes * 8 * case["state"]
        if case.get("packed"):
            total += case["batch"] * case["seq"]
        return {"bytes": total, "flops": n * (75 if grad else 35)}
    if case["kind"] == "norm":
        n, d = case["rows"] * case["width"], case["width"]
        values = 4 + case["gate"] + (4 + case["gate"] if case["grad"] else 0)
        weights = (2 + case["post"]) * (2 if case["grad"] else 1)
        return {"bytes": n * e * values + d * 4 * weights, "flops": n * (45 if case["grad"] else 18)}
    n = sum(_sizes(case))
    states = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": n * (3 * e + states), "flops": n * (15 if case["bits"] == 32 else 60)}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] in ("scan", "step"):
            return _scan_exact(s)
        return _norm_exact(s) if case["kind"] == "norm" else _adamw_exact(s)


def _scan_exact(s):
    """The recurrence token by token."""
    c = s["case"]
    dt, g, x, lam = (s[k].detach().double() for k in ("dt", "g", "x", "log_rate"))
    batch, seq, width = x.shape
    delta = torch.logaddexp(dt, torch.zeros_like(dt))
    p = delta * lam.exp()
    a, sig = (-p).exp(), torch.sigmoid(g)
    cut = s.get("reset")
    h = x.new_zeros(batch, width) if s["h0"] is None else s["h0"].detach().double()
    before, after = [], []
    for t in range(seq):
        if cut is not None:
            h = torch.where(cut[:, t, None], 0.0, h)
        before.append(h)
        h = torch.lerp(sig[:, t] * x[:, t], h, a[:, t])
        after.append(h)
    out = {"y": torch.stack(after, 1), "h": h}
    if not c.get("grad"):
        return out
    dp, ds = torch.empty_like(p), torch.empty_like(p)
    bar = x.new_zeros(batch, width) if s["dh"] is None else s["dh"].double()
    for t in reversed(range(seq)):
        bar = bar + s["dy"][:, t].double()
        dp[:, t] = bar * a[:, t] * (sig[:, t] * x[:, t] - before[t])
        ds[:, t] = bar * -torch.expm1(-p[:, t])
        bar = bar * a[:, t]
        if cut is not None:
            bar = torch.where(cut[:, t, None], 0.0, bar)
    out |= {"ddt": dp * lam.exp() * torch.sigmoid(dt), "dg": ds * x * sig * torch.sigmoid(-g),
            "dx": ds * sig, "dlog_rate": (dp * p).sum((0, 1))}
    if s["h0"] is not None:
        out["dh0"] = bar
    return out


def _norm_exact(s):
    """Values from the definition, gradients by differentiating it."""
    leaves = {k: s[k].detach().double().requires_grad_(s["case"]["grad"])
              for k in ("x", "y", "z", "post", "scale", "pre") if s[k] is not None}
    with torch.set_grad_enabled(s["case"]["grad"]):
        r = leaves["y"]
        if "z" in leaves:
            r = torch.sigmoid(leaves["z"]) * r
        if "post" in leaves:
            r = leaves["post"] * r / (r.square().mean(1, keepdim=True) + NORM_EPS).sqrt()
        out = leaves["x"] + leaves["scale"] * r
        n = leaves["pre"] * out / (out.square().mean(1, keepdim=True) + NORM_EPS).sqrt()
        got = {"out": out.detach(), "n": n.detach()}
        if s["case"]["grad"]:
            grads = torch.autograd.grad([out, n], list(leaves.values()),
                                        [s["dout"].double(), s["dn"].double()])
            got |= {"d" + k: v for k, v in zip(leaves, grads)}
    return got


def _adamw_exact(s):
    """The 8-bit states as what their codes stand for before rounding, in units of the scale."""
    c = s["case"]
    t = s["step"] + 1
    p, g = s["p"].double(), s["grad"].double()
    norm = torch.linalg.vector_norm(g)
    if c["clip"]:
        g = g * min(1.0, MAX_NORM / (norm.item() + 1e-6))
    if c["bits"] == 32:
        m, v = s["m"].double(), s["v"].double()
    else:
        m = s["m"].double() * s["m_scale"].double().repeat_interleave(BLOCK)
        v = (s["v"].double() * s["v_scale"].double().repeat_interleave(BLOCK)) ** 2
    m = torch.lerp(g, m, BETA1)
    v = torch.lerp(g * g, v, BETA2)
    hat = (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + ADAM_EPS)
    out = {"p": p - LR * (hat + DECAY * p), "m": m, "v": v, "norm": norm if c["clip"] else None}
    if c["bits"] == 8:
        for name, value in (("m", m), ("v", v.sqrt())):
            top = value.view(-1, BLOCK).abs().amax(1)
            scale = torch.exp2(torch.ceil(torch.log2(top.clamp_min(2.0 ** -117) / 448)).clamp_min(-126))
            scale = torch.where(top == 0, 2.0 ** -126, scale)
            out[name + "_scale"] = scale
            out[name] = value / scale.repeat_interleave(BLOCK)
    return out
