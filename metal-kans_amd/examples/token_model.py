"""Trains a small next-token model of Chebyshev KAN layers on one MI355X.

The blocks are ``TorchMetalKANLinear`` pairs; around them run ``embedding`` (the tokens' rows),
``dropout``, ``residual_norm`` (the norms, gates and residual scale between blocks), ``linear_cross_entropy`` (the loss
under the vocabulary's head, without its logits) and ``TorchAdamW`` (states in 8 or 32 bits).  What a token knows of those
before it is the row of the one before (``--mixer pair``) or comes through a ``causal_conv`` and a ``selective_scan`` in front of
every block (``--mixer scan``), which then also serve: a prompt, and one token after the other, from the
states that they carry.  The data is synthetic: each token is a fixed function of the two before it, with some noise, and
padding at the ends of the sequences.

    python metal-kans_amd/examples/token_model.py --steps 200
    python metal-kans_amd/examples/token_model.py --steps 200 --mixer scan --dropout 0.1
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


class ScanMixer(nn.Module):
    """Mixes along the sequence: a projection's one half through a short convolution and a scan, gated by the other."""

    def __init__(self, width: int, states: int = 8, taps: int = 4, rank: int = 8):
        super().__init__()
        self.states, self.rank = states, rank
        self.inside = nn.Linear(width, 2 * width, bias=False)
        self.taps = nn.Parameter(torch.randn(width, taps) / taps ** 0.5)
        self.taps_bias = nn.Parameter(torch.zeros(width))
        self.select = nn.Linear(width, rank + 2 * states, bias=False)
        self.step = nn.Linear(rank, width, bias=False)
        self.step_bias = nn.Parameter(torch.log(torch.expm1(torch.exp(torch.empty(width).uniform_(np.log(0.01), np.log(0.3))))))
        self.decay = nn.Parameter(torch.log(torch.arange(1.0, states + 1)).repeat(width, 1))
        self.skip = nn.Parameter(torch.ones(width))
        self.outside = nn.Linear(width, width, bias=False)

    def start(self, rows: int):
        """The states before the first token: of the convolution, of the scan."""
        width, taps = self.taps.shape
        return (torch.zeros(rows, taps - 1, width, device=self.taps.device),
                torch.zeros(rows, width, self.states, device=self.taps.device))

    def forward(self, h: torch.Tensor, carried=(None, None)) -> torch.Tensor:
        x, gate = self.inside(h).chunk(2, -1)
        x = mk.causal_conv(x, self.taps, self.taps_bias, state=carried[0])
        step, b, c = self.select(x).split([self.rank, self.states, self.states], -1)
        y = mk.selective_scan(x, self.step(step), -torch.exp(self.decay), b, c, D=self.skip, z=gate, dt_bias=self.step_bias,
                              state=carried[1])
        return self.outside(y)


class TokenModel(nn.Module):
    """Tokens -> hidden rows; the head is applied by the loss."""

    def __init__(self, vocab: int, width: int, blocks: int, degree: int = 4, mixer: str = "pair", dropout: float = 0.0):
        super().__init__()
        self.dropout, self.seed = dropout, None   # (a one-element int64 tensor where dropout is on)
        self.embed = nn.Parameter(0.3 * torch.randn(2, vocab, width))
        self.blocks = nn.ModuleList(nn.Sequential(mk.TorchMetalKANLinear(width, 2 * width, degree=degree),
                                                  mk.TorchMetalKANLinear(2 * width, width, degree=degree))
                                    for _ in range(blocks))
        ones = lambda: nn.ParameterList([nn.Parameter(torch.ones(width)) for _ in range(blocks + 1)])  # noqa: E731
        self.pre, self.post, self.gate = ones(), ones(), ones()
        self.scale = nn.ParameterList([nn.Parameter(torch.full((1,), 0.5)) for _ in range(blocks)])
        self.head = nn.Parameter(torch.randn(vocab, width) / width ** 0.5)
        self.mixers = nn.ModuleList(ScanMixer(width) for _ in range(blocks)) if mixer == "scan" else None

    def drop(self, x: torch.Tensor, place: int) -> torch.Tensor:
        return x if self.seed is None else mk.dropout(x, self.dropout, self.seed, offset=place)

    def start(self, rows: int):
        """The states of every mixer before the first token."""
        return [m.start(rows) for m in self.mixers]

    def forward(self, tokens: torch.Tensor, carried=None) -> torch.Tensor:
        x = mk.embedding(tokens, self.embed[0])
        if self.mixers is None:
            before = torch.cat([tokens[:, :1], tokens[:, :-1]], 1)
            x = x + mk.embedding(before, self.embed[1])
        x = self.drop(x, 0)
        x, h = mk.residual_norm(x, pre_weight=self.pre[0], kind="layer")
        for i, block in enumerate(self.blocks):
            if self.mixers is not None:
                h = h + self.mixers[i](h, carried[i] if carried else (None, None))
            x, h = mk.residual_norm(x, self.drop(block(torch.tanh(h)), i + 1), gate=self.gate[i], scale=self.scale[i],
                                    post_weight=self.post[i], pre_weight=self.pre[i + 1], kind="layer")
        return h

    @torch.no_grad()
    def generate(self, tokens: torch.Tensor, count: int) -> torch.Tensor:
        """The most likely next `count` tokens behind prompts [rows, length]: the prompt once, then a token at a time."""
        carried, out = self.start(tokens.shape[0]), []
        for _ in range(count):
            h = self.forward(tokens, carried)
            tokens = (h[:, -1:] @ self.head.t()).argmax(-1)
            out.append(tokens)
        return torch.cat(out, 1)


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
          state_bits: int = 8, seed: int = 0, quiet: bool = False, mixer: str = "pair", dropout: float = 0.0):
    """The losses of the steps."""
    torch.manual_seed(seed)
    np.random.seed(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    model = TokenModel(vocab, width, blocks, mixer=mixer, dropout=dropout).cuda()
    if dropout:
        model.seed = torch.zeros(1, dtype=torch.int64, device="cuda")
    opt = mk.TorchAdamW(model.parameters(), lr=3e-3, weight_decay=0.01, state_bits=state_bits)
    losses = []
    start = time.perf_counter()
    for step in range(steps):
        tokens, target = batch(gen, rows, length, vocab)
        loss = mk.linear_cross_entropy(model(tokens), model.head, target, ignore_index=IGNORE)
        opt.zero_grad()
        loss.backward()
        if dropout:
            model.seed += 1
        opt.step()
        losses.append(loss.detach())
        if not quiet and (step + 1) % 20 == 0:
            print(f"step {step + 1}: loss {loss.item():.3f}, {(time.perf_counter() - start) / (step + 1) * 1e3:.2f} ms a step",
                  flush=True)
    if mixer == "scan" and not quiet:
        model.seed = None
        tokens, target = batch(gen, 8, length, vocab)
        half = length // 2
        right = model.generate(tokens[:, :half], 1)[:, 0] == target[:, half - 1]
        print(f"next token of {half}: {right.sum().item()} of 8 as in the data")
    return torch.stack(losses).tolist()


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--width", type=int, default=64)
    ap.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    ap.add_argument("--mixer", default="pair", choices=("pair", "scan"))
    ap.add_argument("--dropout", type=float, default=0.0)
    a = ap.parse_args()
    train(steps=a.steps, width=a.width, state_bits=a.state_bits, mixer=a.mixer, dropout=a.dropout)
