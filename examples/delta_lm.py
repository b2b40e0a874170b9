"""A small language model of gated delta rules, trained and sampled with the framework's operators: layer
norm, the rule over packed documents (in sampling one token at a time), Muon for the layers' matrices and
AdamW for all else.

    python examples/delta_lm.py [--steps 200] [--dtype bf16]

The data are those of gated_lm.py: documents of a random Markov chain, packed into rows without padding.
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch
import torch.nn as nn
import torch.nn.functional as F

sys.path[:0] = [str(Path(__file__).resolve().parents[1]), str(Path(__file__).resolve().parent)]

from gated_lm import documents  # noqa: E402
from mambaqc_amd.kernels import gated_delta, gated_delta_step_  # noqa: E402
from mambaqc_amd.layers import LayerNorm  # noqa: E402
from mambaqc_amd.optim import AdamW, Muon  # noqa: E402


class DeltaLayer(nn.Module):
    """One projection makes queries and keys (shared by `group` value heads each), values, and both gates."""

    def __init__(self, d_model: int, heads: int, group: int, k_dim: int, v_dim: int):
        super().__init__()
        self.heads, self.k_dim, self.v_dim = heads, k_dim, v_dim
        self.values = heads * group
        self.sizes = [heads * k_dim, heads * k_dim, self.values * v_dim]
        self.norm = LayerNorm(d_model)
        self.proj = nn.Linear(d_model, sum(self.sizes), bias=False)
        self.gates = nn.Linear(d_model, 2 * self.values)
        self.out_norm = LayerNorm(v_dim)
        self.out = nn.Linear(self.values * v_dim, d_model, bias=False)
        # Heads that forget within a few tokens to ones that hold for thousands.
        self.log_rate = nn.Parameter(torch.linspace(math.log(1e-3), math.log(0.5), self.values))

    def forward(self, stream, reset=None, h=None):
        """(the stream after the layer, the state); h is updated in place for one token without gradients
        and reset."""
        n = self.norm(stream)
        q, k, v = self.proj(n).split(self.sizes, -1)
        q, k = (F.normalize(x.unflatten(-1, (self.heads, self.k_dim)).float(), dim=-1).to(v.dtype)
                for x in (q, k))
        v = v.unflatten(-1, (self.values, self.v_dim))
        decay, beta = self.gates(n).float().chunk(2, -1)
        decay, beta = -F.softplus(decay) * self.log_rate.float().exp(), beta.sigmoid()
        if h is not None and n.shape[1] == 1 and reset is None and not torch.is_grad_enabled():
            o = gated_delta_step_(q, k, v, decay, beta, h)
        else:
            o, h = gated_delta(q, k, v, decay, beta, h0=h, reset=reset, return_state=True)
        return stream + self.out(self.out_norm(o).flatten(2)), h


class DeltaLM(nn.Module):
    def __init__(self, vocab: int, d_model: int = 128, heads: int = 2, group: int = 2, k_dim: int = 32,
                 v_dim: int = 64, layers: int = 2):
        super().__init__()
        self.embedding = nn.Embedding(vocab, d_model)
        self.layers = nn.ModuleList(DeltaLayer(d_model, heads, group, k_dim, v_dim) for _ in range(layers))
        self.norm = LayerNorm(d_model)
        self.head = nn.Linear(d_model, vocab, bias=False)

    def forward(self, tokens, reset=None, states=None):
        """(logits, the layers' states)."""
        stream, after = self.embedding(tokens), []
        for layer, h in zip(self.layers, states or [None] * len(self.layers)):
            stream, h = layer(stream, reset, h)
            after.append(h)
        return self.head(self.norm(stream)), after

    @torch.no_grad()
    def generate(self, prompt, count: int):
        """`count` more tokens for each row, the likeliest ones: the prompt once, then a step each."""
        out, states = [prompt], None
        for _ in range(count):
            logits, states = self(out[-1], states=states)
            out.append(logits[:, -1:].argmax(-1))
        return torch.cat(out, 1)

    def optimizers(self):
        """Muon for the layers' projections; AdamW for embedding, head, gates and norms."""
        matrices = [w for layer in self.layers for w in (layer.proj.weight, layer.out.weight)]
        ids = {id(w) for w in matrices}
        others = [p for p in self.parameters() if id(p) not in ids]
        return [Muon(matrices, lr=0.02, weight_decay=0.01),
                AdamW(others, lr=3e-3, betas=(0.9, 0.95), weight_decay=0.01)]


def loss_of(model, tokens, start):
    """The mean loss of packed documents, tokens [batch, length + 1] with `start` true at first tokens."""
    logits, _ = model(tokens[:, :-1], reset=start[:, :-1])
    # (a document's first token does not follow from the one before it)
    target = tokens[:, 1:].masked_fill(start[:, 1:], -100)
    return F.cross_entropy(logits.float().flatten(0, 1), target.flatten(), ignore_index=-100)


def train(model, steps: int, batch: int = 8, length: int = 128, seed: int = 0, report=None):
    """The losses of `steps` steps, and the chain's table."""
    gen = torch.Generator().manual_seed(seed)
    vocab, device = model.embedding.num_embeddings, model.embedding.weight.device
    table = torch.randperm(vocab, generator=gen)
    optimizers = model.optimizers()
    losses = []
    for step in range(steps):
        tokens, start = (t.to(device) for t in documents(gen, table, batch, length))
        for optimizer in optimizers:
            optimizer.zero_grad()
        loss = loss_of(model, tokens, start)
        loss.backward()
        for optimizer in optimizers:
            optimizer.step()
        losses.append(loss.detach())
        if report and (step % 20 == 0 or step == steps - 1):
            report(f"step {step:4d}  loss {loss.item():.3f}")
    return [v.item() for v in losses], table


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    parser.add_argument("--steps", type=int, default=200)
    parser.add_argument("--dtype", default="fp32", choices=("fp32", "bf16"))
    args = parser.parse_args()
    torch.manual_seed(0)
    model = DeltaLM(64).to("cuda", torch.bfloat16 if args.dtype == "bf16" else torch.float32)
    _, table = train(model, args.steps, report=print)
    out = model.generate(torch.arange(8, device="cuda")[:, None], 16).cpu()
    right = (out[:, 1:] == table[out[:, :-1]]).float().mean().item()
    print(f"of 16 tokens sampled after each of 8, {100 * right:.0f} % follow the chain")


if __name__ == "__main__":
    main()
