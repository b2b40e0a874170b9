"""The recurrent operators together, as examples/gated_lm.py trains and samples with them."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
spec = importlib.util.spec_from_file_location(
    "gated_lm", Path(__file__).resolve().parents[1] / "examples" / "gated_lm.py")
gated_lm = importlib.util.module_from_spec(spec)
spec.loader.exec_module(gated_lm)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 32])
def test_trains_and_samples(dtype, bits):
    """The chain gives 0.1 log 64 + the entropy of (0.9, 0.1), 0.74 nats a token, the unigram 4.16:
    after 120 steps the loss is below half of that, and what is sampled mostly follows the chain."""
    torch.manual_seed(0)
    model = gated_lm.GatedLM(64, d_model=64, width=96).to(DEV, dtype)
    losses, table = gated_lm.train(model, 120, bits)
    assert losses[0] > 3.5 and sum(losses[-10:]) / 10 < 2.08
    out = model.generate(torch.arange(16, device=DEV)[:, None], 12).cpu()
    assert (out[:, 1:] == table[out[:, :-1]]).float().mean() > 0.6


def test_steps_are_the_whole_forward():
    """Logits token by token equal those of one forward; packed documents equal each alone."""
    torch.manual_seed(1)
    model = gated_lm.GatedLM(50, d_model=48, width=80).to(DEV)
    tokens = torch.randint(50, (3, 40), device=DEV)
    with torch.no_grad():
        whole, ends = model(tokens)
        got, states = model(tokens[:, :7])
        parts = [got]
        for t in range(7, 40):
            got, states = model(tokens[:, t:t + 1], states=states)
            parts.append(got)
        # fp32 products of a few hundred terms on either side: 2^-14 of logits of about 1.
        assert (torch.cat(parts, 1) - whole).abs().max() < 2.0 ** -14
        for a, b in zip(states, ends):
            assert (a - b).abs().max() < 2.0 ** -14
        reset = torch.zeros(3, 40, dtype=torch.bool, device=DEV)
        reset[:, 25] = True
        packed, _ = model(tokens, reset=reset)
        alone, _ = model(tokens[:, 25:])
        assert (packed[:, 25:] - alone).abs().max() < 2.0 ** -14
        assert (packed[:, :25] - whole[:, :25]).abs().max() < 2.0 ** -14


def test_one_token_that_starts_a_document():
    """A reset at a single token counts, with a state in hand and without gradients."""
    torch.manual_seed(2)
    model = gated_lm.GatedLM(50, d_model=48, width=80).to(DEV)
    tokens = torch.randint(50, (2, 9), device=DEV)
    with torch.no_grad():
        _, states = model(tokens[:, :8])
        fresh, _ = model(tokens[:, 8:])
        reset = torch.tensor([[True], [False]], device=DEV)
        got, _ = model(tokens[:, 8:], reset=reset, states=[h.clone() for h in states])
        whole, _ = model(tokens)
    assert (got[0] - fresh[0]).abs().max() < 2.0 ** -14
    assert (got[1] - whole[1, 8:]).abs().max() < 2.0 ** -14
    assert (fresh[1] - whole[1, 8:]).abs().max() > 2.0 ** -10  # (the state matters)
