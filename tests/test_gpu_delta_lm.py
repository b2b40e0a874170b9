"""Layer norm, the gated delta rule, its step and Muon together, as examples/delta_lm.py uses them."""
import importlib.util
from pathlib import Path

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda"
spec = importlib.util.spec_from_file_location(
    "delta_lm", Path(__file__).resolve().parents[1] / "examples" / "delta_lm.py")
delta_lm = importlib.util.module_from_spec(spec)
spec.loader.exec_module(delta_lm)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_trains_and_samples(dtype):
    torch.manual_seed(0)
    model = delta_lm.DeltaLM(64, d_model=64, v_dim=48).to(DEV, dtype)
    before = {k: v.clone() for k, v in model.state_dict().items()}
    losses, table = delta_lm.train(model, 12)
    assert all(torch.isfinite(torch.tensor(losses)))
    for name, p in model.named_parameters():
        assert p.isfinite().all(), name
        # (AdamW's step of at most about 3e-3 is less than half a bf16 spacing, 2^-7 or more, at log_rate's
        # values beyond 2: it may round to nothing there)
        if dtype == torch.float32 or not name.endswith("log_rate"):
            assert not torch.equal(p, before[name]), name
    out = model.generate(torch.arange(16, device=DEV)[:, None], 12)
    assert out.shape == (16, 13) and int(out.min()) >= 0 and int(out.max()) < 64


def test_steps_are_the_whole_forward():
    """Logits token by token equal those of one forward; packed documents equal each alone."""
    torch.manual_seed(1)
    model = delta_lm.DeltaLM(50, d_model=48, v_dim=40).to(DEV)
    tokens = torch.randint(50, (3, 90), device=DEV)
    with torch.no_grad():
        whole, ends = model(tokens)
        got, states = model(tokens[:, :70])
        parts = [got]
        for t in range(70, 90):
            got, states = model(tokens[:, t:t + 1], states=states)
            parts.append(got)
        # fp32 products of a few hundred terms on either side: 2^-14 of logits of about 1.
        assert (torch.cat(parts, 1) - whole).abs().max() < 2.0 ** -14
        for a, b in zip(states, ends):
            assert (a - b).abs().max() < 2.0 ** -14
        reset = torch.zeros(3, 90, dtype=torch.bool, device=DEV)
        reset[:, 25] = True
        packed, _ = model(tokens, reset=reset)
        alone, _ = model(tokens[:, 25:])
        assert (packed[:, 25:] - alone).abs().max() < 2.0 ** -14
        assert (packed[:, :25] - whole[:, :25]).abs().max() < 2.0 ** -14
        assert (packed[:, 25:] - whole[:, 25:]).abs().max() > 2.0 ** -10  # (the reset matters)


def test_one_token_that_starts_a_document():
    """A reset at a single token counts, with a state in hand and without gradients."""
    torch.manual_seed(2)
    model = delta_lm.DeltaLM(50, d_model=48, v_dim=40).to(DEV)
    tokens = torch.randint(50, (2, 9), device=DEV)
    with torch.no_grad():
        _, states = model(tokens[:, :8])
        fresh, _ = model(tokens[:, 8:])
        reset = torch.tensor([[True], [False]], device=DEV)
        got, _ = model(tokens[:, 8:], reset=reset, states=[h.clone() for h in states])
        whole, _ = model(tokens)
    assert (got[0] - fresh[0]).abs().max() < 2.0 ** -14
    assert (got[1] - whole[1, 8:]).abs().max() < 2.0 ** -14


def plain_loss(model, w, tokens, start):
    """The example's loss from its formulas, parameters `w` in 64 bits, a token at a time."""
    stream = w["embedding.weight"][tokens[:, :-1]]
    b, t, d = stream.shape
    for i, layer in enumerate(model.layers):
        def p(name):
            return w[f"layers.{i}.{name}"]
        n = F.layer_norm(stream, (d,), p("norm.weight"), p("norm.bias"))
        q, k, v = (n @ p("proj.weight").T).split(layer.sizes, -1)
        q, k = (F.normalize(x.unflatten(-1, (layer.heads, layer.k_dim)), dim=-1)
                .repeat_interleave(layer.values // layer.heads, 2) for x in (q, k))
        v = v.unflatten(-1, (layer.values, layer.v_dim))
        decay, beta = (n @ p("gates.weight").T + p("gates.bias")).chunk(2, -1)
        keep, beta = (-F.softplus(decay) * p("log_rate").exp()).exp(), beta.sigmoid()
        S, o = torch.zeros(b, layer.values, layer.k_dim, layer.v_dim, dtype=torch.float64), []
        for j in range(t):
            S = S * (keep[:, j] * ~start[:, j, None])[..., None, None]
            r = beta[:, j, :, None] * (v[:, j] - (k[:, j, :, :, None] * S).sum(2))
            S = S + k[:, j, :, :, None] * r[:, :, None]
            o.append((q[:, j, :, :, None] * S).sum(2) * layer.k_dim ** -0.5)
        o = F.layer_norm(torch.stack(o, 1), (layer.v_dim,), p("out_norm.weight"), p("out_norm.bias"))
        stream = stream + o.flatten(2) @ p("out.weight").T
    logits = F.layer_norm(stream, (d,), w["norm.weight"], w["norm.bias"]) @ w["head.weight"].T
    target = tokens[:, 1:].masked_fill(start[:, 1:], -100)
    return F.cross_entropy(logits.flatten(0, 1), target.flatten(), ignore_index=-100)


def test_gradients():
    """Against the formulas in 64 bits, and their sum along a direction against differences of the loss."""
    torch.manual_seed(3)
    model = delta_lm.DeltaLM(20, d_model=24, heads=2, group=2, k_dim=9, v_dim=13).to(DEV)
    tokens, start = delta_lm.documents(torch.Generator().manual_seed(4), torch.randperm(20), 3, 75)
    loss = delta_lm.loss_of(model, tokens.to(DEV), start.to(DEV))
    loss.backward()
    w = {k: v.detach().double().cpu().requires_grad_() for k, v in model.named_parameters()}
    want = plain_loss(model, w, tokens, start)
    want.backward()
    # fp32 sums of a few hundred terms through two layers, as above: 2^-14 of the largest.
    assert abs(loss.item() - want.item()) < 2.0 ** -14 * want.item()
    got = {k: p.grad.double().cpu() for k, p in model.named_parameters()}
    for k, p in w.items():
        assert (got[k] - p.grad).abs().max() <= 2.0 ** -14 * p.grad.abs().max(), k
    # A central difference over 2^-12 (its third-order term: 2^-24 of derivatives of about 1).
    gen = torch.Generator().manual_seed(5)
    way = {k: torch.randn(p.shape, generator=gen, dtype=torch.float64) / p.numel() ** 0.5
           for k, p in w.items()}
    with torch.no_grad():
        up, down = (plain_loss(model, {k: p + s * way[k] for k, p in w.items()}, tokens, start)
                    for s in (2.0 ** -12, -2.0 ** -12))
    slope = sum((got[k] * way[k]).sum() for k in w)
    size = sum((got[k] * way[k]).abs().sum() for k in w)
    assert abs((up - down) * 2.0 ** 11 - slope) <= 2.0 ** -14 * size
