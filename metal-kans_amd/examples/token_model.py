"""Trains a small next-token model of Chebyshev KAN layers on one MI355X.

The blocks are ``TorchMetalKANLinear`` pairs; around them run ``residual_norm`` (the norms, gates and residual
scale between blocks), ``linear_cross_entropy`` (the loss under the vocabulary's head, without its logits) and
``TorchAdamW`` (states in 8 or 32 bits).  The data is synthetic: each token is a fixed function of the two
before it, with some noise, and padding at the ends of the sequences.

    python metal-kans_amd/examples/token_model.py --steps 200
"""
import argparse
import os
import sys
import time

import numpy as np
import torch
import torch.nn as nn

sys.path.insert(0, os.path.abspath(os.path.join(os.path.dirname(__file__), "..")))

import metal_kans as mk  # noqa: E402

IGNORE = -100


class TokenModel(nn.Module):
    """Token pairs -> hidden rows; the head is applied by the loss."""

    def __init__(self, vocab: int, width: int, blocks: int, degree: int = 4):
        super().__init__()
        self.embed = nn.Parameter(0.3 * torch.randn(2, vocab, width))
        self.blocks = nn.ModuleList(nn.Sequential(mk.TorchMetalKANLinear(width, 2 * width, degree=degree),
                                                  mk.TorchMetalKANLinear(2 * width, width, degree=degree))
                                    for _ in range(blocks))
        ones = lambda: nn.ParameterList([nn.Parameter(torch.ones(width)) for _ in range(blocks + 1)])  # noqa: E731
        self.pre, self.post, self.gate = ones(), ones(), ones()
        self.scale = nn.ParameterList([nn.Parameter(torch.full((1,), 0.5)) for _ in range(blocks)])
        self.head = nn.Parameter(torch.randn(vocab, width) / width ** 0.5)

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        before = torch.cat([tokens[:, :1], tokens[:, :-1]], 1)
        x = self.embed[0][tokens] + self.embed[1][before]
        x, h = mk.residual_norm(x, pre_weight=self.pre[0], kind="layer")
        for i, block in enumerate(self.blocks):
            x, h = mk.residual_norm(x, block(torch.tanh(h)), gate=self.gate[i], scale=self.scale[i],
                                    post_weight=self.post[i], pre_weight=self.pre[i + 1], kind="layer")
        return h


def batch(gen: torch.Generator, rows: int, length: int, vocab: int):
    """Tokens and their successors; the last part of every other sequence is padding."""
    t = torch.randint(0, vocab, (rows, length + 1), generator=gen, device="cuda")
    for i in range(2, length + 1):
        t[:, i] = (3 * t[:, i - 1] + 5 * t[:, i - 2] + 1) % vocab
    noise = torch.rand(t.shape, generator=gen, device="cuda") < 0.05
    t = torch.where(noise, torch.randint(0, vocab, t.shape, generator=gen, device="cuda"), t)
    target = t[:, 1:].clone()
    target[::2, length - length // 4:] = IGNORE
    return t[:, :-1], target


def train(steps: int = 200, vocab: int = 61, width: int = 64, blocks: int = 2, rows: int = 64, length: int = 32,
          state_bits: int = 8, seed: int = 0, quiet: bool = False):
    """The losses of the steps."""
    torch.manual_seed(seed)
    np.random.seed(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    model = TokenModel(vocab, width, blocks).cuda()
    opt = mk.TorchAdamW(model.parameters(), lr=3e-3, weight_decay=0.01, state_bits=state_bits)
    losses = []
    start = time.perf_counter()
    for step in range(steps):
        tokens, target = batch(gen, rows, length, vocab)
        loss = mk.linear_cross_entropy(model(tokens), model.head, target, ignore_index=IGNORE)
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
        if not quiet and (step + 1) % 20 == 0:
            print(f"step {step + 1}: loss {loss.item():.3f}, {(time.perf_counter() - start) / (step + 1) * 1e3:.2f} ms a step",
                  flush=True)
    return torch.stack(losses).tolist()


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--width", type=int, default=64)
    ap.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    a = ap.parse_args()
    train(steps=a.steps, width=a.width, state_bits=a.state_bits)
