"""examples/delta_lm.py without a GPU: how many tokens are sampled, and which optimiser has what."""
import importlib.util
from pathlib import Path

import pytest
import torch

spec = importlib.util.spec_from_file_location(
    "delta_lm", Path(__file__).resolve().parents[1] / "examples" / "delta_lm.py")
delta_lm = importlib.util.module_from_spec(spec)
spec.loader.exec_module(delta_lm)


@pytest.mark.parametrize("count", [0, 1, 2, 5])
def test_generate_samples_as_many_as_asked(count, monkeypatch):
    """Against a forward that says the next number, and that sees the prompt once, then single tokens."""
    seen = []

    def forward(self, tokens, reset=None, states=None):
        seen.append((tuple(tokens.shape), states))
        return torch.nn.functional.one_hot((tokens + 1) % 11, 11).float(), len(seen)

    monkeypatch.setattr(delta_lm.DeltaLM, "forward", forward)
    prompt = torch.tensor([[4, 2, 7], [0, 1, 2]])
    got = delta_lm.DeltaLM(11, d_model=4, heads=1, k_dim=4, v_dim=4, layers=1).generate(prompt, count)
    want = torch.stack([(prompt[:, -1] + i) % 11 for i in range(1, count + 1)], 1) if count else prompt[:, :0]
    assert torch.equal(got, torch.cat([prompt, want], 1))
    assert seen == [((2, 1 if i else 3), i or None) for i in range(count)]


def test_every_parameter_has_one_optimiser():
    model = delta_lm.DeltaLM(11, d_model=8, heads=1, k_dim=4, v_dim=4, layers=2)
    muon, adamw = model.optimizers()
    has = [p for opt in (muon, adamw) for g in opt.param_groups for p in g["params"]]
    assert sorted(map(id, has)) == sorted(map(id, model.parameters()))
    assert all(p.dim() == 2 for g in muon.param_groups for p in g["params"])
