"""A small language model of gated scans, trained and sampled with the framework's recurrent operators:
the scan (packed documents in training, one token at a time in sampling), the gate with norms and
residual between its layers, and AdamW with its states in 8 or in 32 bits.

    python examples/gated_lm.py [--steps 200] [--state-bits 8] [--dtype bf16]

The data are documents of a random Markov chain, packed into rows without padding.
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from mambaqc_amd.kernels import gate_norm_residual, gated_scan, gated_scan_step_  # noqa: E402
from mambaqc_amd.optim import AdamW  # noqa: E402


class GatedLayer(nn.Module):
    """One projection makes the scan's step, gate and input and the output's gate; the scan walks them."""

    def __init__(self, d_model: int, width: int):
        super().__init__()
        self.width = width
        self.proj = nn.Linear(d_model, 3 * width + d_model, bias=False)
        self.out = nn.Linear(width, d_model, bias=False)
        # Channels that forget within a token to ones that hold for thousands.
        self.log_rate = nn.Parameter(torch.linspace(math.log(1e-3), math.log(2.0), width))
        self.post = nn.Parameter(torch.ones(d_model))
        self.scale = nn.Parameter(torch.full((d_model,), 0.5))
        self.pre = nn.Parameter(torch.ones(d_model))

    def forward(self, stream, n, reset=None, h=None):
        """(the stream after the layer, the next one's input, the state); h is updated in place for
        one token without gradients and reset."""
        w = self.width
        dt, g, x, z = self.proj(n).split([w, w, w, n.shape[-1]], -1)
        if h is not None and n.shape[1] == 1 and reset is None and not torch.is_grad_enabled():
            y = gated_scan_step_(dt, g, x, self.log_rate, h)
        else:
            y, h = gated_scan(dt, g, x, self.log_rate, h0=h, reset=reset, return_state=True)
        stream, n = gate_norm_residual(stream, self.out(y), z, post_weight=self.post,
                                       scale=self.scale, pre_weight=self.pre)
        return stream, n, h


class GatedLM(nn.Module):
    def __init__(self, vocab: int, d_model: int = 128, width: int = 256, layers: int = 2):
        super().__init__()
        self.embedding = nn.Embedding(vocab, d_model)
        self.norm = nn.RMSNorm(d_model, eps=1e-6)
        self.layers = nn.ModuleList(GatedLayer(d_model, width) for _ in range(layers))
        self.head = nn.Linear(d_model, vocab, bias=False)

    def forward(self, tokens, reset=None, states=None):
        """(logits, the layers' states)."""
        stream = self.embedding(tokens)
        n, after = self.norm(stream), []
        for layer, h in zip(self.layers, states or [None] * len(self.layers)):
            stream, n, h = layer(stream, n, reset, h)
            after.append(h)
        return self.head(n), after

    @torch.no_grad()
    def generate(self, prompt, count: int):
        """`count` more tokens for each row, the likeliest ones: the prompt once, then a step each."""
        out, states = [prompt], None
        for _ in range(count):
            logits, states = self(out[-1], states=states)
            out.append(logits[:, -1:].argmax(-1))
        return torch.cat(out, 1)


def documents(gen, table, batch: int, length: int):
    """Rows of packed documents (tokens [batch, length + 1], true at each document's first token): a
    token is the one that `table` has for the token before it nine times out of ten."""
    vocab = table.numel()
    start = torch.rand(batch, length + 1, generator=gen) < 1 / 24
    start[:, 0] = True
    free = start | (torch.rand(batch, length + 1, generator=gen) < 0.1)
    tokens = torch.randint(vocab, (batch, length + 1), generator=gen)
    for t in range(1, length + 1):
        tokens[:, t] = torch.where(free[:, t], tokens[:, t], table[tokens[:, t - 1]])
    return tokens, start


def train(model, steps: int, state_bits: int = 8, batch: int = 8, length: int = 128, seed: int = 0,
          report=None):
    """The losses of `steps` steps, and the chain's table."""
    gen = torch.Generator().manual_seed(seed)
    vocab, device = model.embedding.num_embeddings, model.embedding.weight.device
    table = torch.randperm(vocab, generator=gen)
    optimizer = AdamW(model.parameters(), lr=3e-3, betas=(0.9, 0.95), weight_decay=0.01,
                      state_bits=state_bits, max_norm=1.0)
    losses = []
    for step in range(steps):
        tokens, start = (t.to(device) for t in documents(gen, table, batch, length))
        optimizer.zero_grad()
        logits, _ = model(tokens[:, :-1], reset=start[:, :-1])
        # (a document's first token does not follow from the one before it)
        target = tokens[:, 1:].masked_fill(start[:, 1:], -100)
        loss = F.cross_entropy(logits.float().flatten(0, 1), target.flatten(), ignore_index=-100)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
        if report and (step % 20 == 0 or step == steps - 1):
            report(f"step {step:4d}  loss {loss.item():.3f}  gradients' norm "
                   f"{optimizer.grad_norm.item():.3f}")
    return [v.item() for v in losses], table


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    parser.add_argument("--dtype", default="fp32", choices=("fp32", "bf16"))
    args = parser.parse_args()
    torch.manual_seed(0)
    model = GatedLM(64).to("cuda", torch.bfloat16 if args.dtype == "bf16" else torch.float32)
    _, table = train(model, args.steps, args.state_bits, report=print)
    out = model.generate(torch.arange(8, device="cuda")[:, None], 16).cpu()
    right = (out[:, 1:] == table[out[:, :-1]]).float().mean().item()
    print(f"of 16 tokens sampled after each of 8, {100 * right:.0f} % follow the chain")


if __name__ == "__main__":
    main()
