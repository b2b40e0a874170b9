"""examples/gated_lm.py without a GPU: how many tokens are sampled."""
import importlib.util
from pathlib import Path

import pytest
import torch

spec = importlib.util.spec_from_file_location(
    "gated_lm", Path(__file__).resolve().parents[1] / "examples" / "gated_lm.py")
gated_lm = importlib.util.module_from_spec(spec)
spec.loader.exec_module(gated_lm)


@pytest.mark.parametrize("count", [0, 1, 2, 5])
def test_generate_samples_as_many_as_asked(count, monkeypatch):
    """Against a forward that says the next number, and that sees the prompt once, then single tokens."""
    seen = []

    def forward(self, tokens, reset=None, states=None):
        seen.append((tuple(tokens.shape), states))
        return torch.nn.functional.one_hot((tokens + 1) % 11, 11).float(), len(seen)

    monkeypatch.setattr(gated_lm.GatedLM, "forward", forward)
    prompt = torch.tensor([[4, 2, 7], [0, 1, 2]])
    got = gated_lm.GatedLM(11, d_model=4, width=4, layers=1).generate(prompt, count)
    want = torch.stack([(prompt[:, -1] + i) % 11 for i in range(1, count + 1)], 1) if count else prompt[:, :0]
    assert torch.equal(got, torch.cat([prompt, want], 1))
    assert seen == [((2, 1 if i else 3), i or None) for i in range(count)]
