"""The token model's operators in one run (on an MI355X): embedding, dropout, causal convolution, selective scan, norms and loss, with
their gradients against the same model on torch's own operations, and the states that serve it."""
import os
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(__file__), "..", "metal-kans_amd", "examples"))


@pytest.fixture(scope="module")
def example(gpu):
    import token_model
    return token_model


def make(example, dropout=0.0, seed=0):
    torch.manual_seed(seed)
    np.random.seed(seed)
    model = example.TokenModel(31, 48, 2, mixer="scan", dropout=dropout).cuda()
    if dropout:
        model.seed = torch.tensor([5], device="cuda")
    return model


class Plain:
    """The operators from torch's operations, under the package's names."""

    def __init__(self, mk):
        self.mk = mk

    def __getattr__(self, name):
        return getattr(self.mk, name)

    def embedding(self, tokens, weight, scale=1.0, ignore_index=-100):
        return scale * torch.nn.functional.embedding(tokens, weight)

    def dropout(self, x, p, seed, offset=0):
        with torch.no_grad():
            kept = self.mk.dropout(torch.ones_like(x), p, seed, offset)
        return x * kept

    def residual_norm(self, x, block=None, gate=None, scale=1.0, post_weight=None, pre_weight=None, kind="rms", eps=1e-6):
        norm = lambda a: torch.nn.functional.layer_norm(a, a.shape[-1:], eps=eps)  # noqa: E731
        if block is not None:
            x = x + scale * gate * (norm(block) * post_weight)
        return x, norm(x) * pre_weight

    def causal_conv(self, x, weight, bias, state=None):
        d, w = weight.shape
        u = torch.nn.functional.conv1d(torch.nn.functional.pad(x.transpose(1, 2), (w - 1, 0)), weight[:, None], bias, groups=d)
        return torch.nn.functional.silu(u.transpose(1, 2))

    def selective_scan(self, x, dt, A, B, C, D, z, dt_bias, state=None):
        s = torch.nn.functional.softplus(dt + dt_bias)
        h, out = 0.0, []
        for t in range(x.shape[1]):
            h = torch.exp(s[:, t, :, None] * A) * h + (s * x)[:, t, :, None] * B[:, t, None]
            out.append((h * C[:, t, None]).sum(-1))
        return (torch.stack(out, 1) + D * x) * torch.nn.functional.silu(z)


@pytest.mark.parametrize("dropout", [0.0, 0.3])
def test_gradients_follow_torch(example, dropout):
    """One loss and its gradients.  fp32 both: within 2e-4 of the largest gradient of each parameter (the layers' own
    bar is 1e-4)."""
    mk = example.mk
    model = make(example, dropout)
    gen = torch.Generator(device="cuda").manual_seed(1)
    tokens, target = example.batch(gen, 8, 40, 31)
    results = []
    for plain in (False, True):
        model.zero_grad(set_to_none=True)
        if plain:
            example.mk = Plain(mk)
        try:
            h = model(tokens)
        finally:
            example.mk = mk
        loss = mk.linear_cross_entropy(h, model.head, target) if not plain else \
            torch.nn.functional.cross_entropy((h @ model.head.t()).flatten(0, 1), target.flatten())
        loss.backward()
        results.append((loss.item(), {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}))
    assert abs(results[0][0] - results[1][0]) <= 1e-5 * abs(results[1][0])
    assert results[0][1].keys() == results[1][1].keys() and len(results[0][1]) > 20
    for n, g in results[0][1].items():
        want = results[1][1][n]
        assert (g - want).abs().max() <= 2e-4 * want.abs().max(), n


def test_states_serve_what_the_whole_sequence_gives(example):
    """A prompt and then single tokens against all tokens at once: fp32 both, and the layers between them to their bar of 1e-4."""
    model = make(example)
    gen = torch.Generator(device="cuda").manual_seed(2)
    tokens, _ = example.batch(gen, 5, 30, 31)
    with torch.no_grad():
        whole = model(tokens)
        carried, at, parts = model.start(5), 0, []
        for n in (17, 1, 1, 1, 3, 1, 1, 1, 1, 1, 1, 1):
            parts.append(model(tokens[:, at:at + n], carried))
            at += n
    assert at == 30
    assert (torch.cat(parts, 1) - whole).abs().max() <= 1e-3 * whole.abs().max()
    out = model.generate(tokens, 4)
    assert out.shape == (5, 4)
    for i in range(4):   # each token from the whole sequence before it
        with torch.no_grad():
            logits = model(tokens)[:, -1] @ model.head.t()
        top, given = logits.max(-1).values, logits.gather(1, out[:, i:i + 1])[:, 0]
        assert ((top - given) <= 1e-3 * logits.abs().max()).all()
        tokens = torch.cat([tokens, out[:, i:i + 1]], 1)


def test_training_runs(example):
    losses = example.train(steps=4, vocab=31, width=48, rows=8, length=24, mixer="scan", dropout=0.1)
    assert len(losses) == 4 and all(np.isfinite(losses))
