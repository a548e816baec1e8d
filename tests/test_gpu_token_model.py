"""The training-step operators together (run on an MI355X): the token model of the examples against the same
model on torch's own operations, and its loss over some steps."""
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


def test_gradients_follow_torch(example):
    """One loss and its gradients: the blocks as they are, the operators around them from torch's operations.
    fp32 both: within 2e-4 of the largest gradient of each parameter (the layers' own bar is 1e-4)."""
    import metal_kans as mk
    torch.manual_seed(0)
    np.random.seed(0)
    model = example.TokenModel(31, 48, 2).cuda()
    gen = torch.Generator(device="cuda").manual_seed(1)
    tokens, target = example.batch(gen, 8, 16, 31)

    def plain_norm(x, block=None, gate=None, scale=1.0, post_weight=None, pre_weight=None, kind="rms", eps=1e-6):
        def norm(a):
            return torch.nn.functional.layer_norm(a, a.shape[-1:], eps=eps)
        if block is not None:
            x = x + scale * gate * (norm(block) * post_weight)
        return x, norm(x) * pre_weight
    results = []
    fused = mk.residual_norm
    for plain in (False, True):
        model.zero_grad(set_to_none=True)
        if plain:
            example.mk.residual_norm = plain_norm
        try:
            h = model(tokens)
        finally:
            example.mk.residual_norm = fused
        loss = mk.linear_cross_entropy(h, model.head, target) if not plain else \
            torch.nn.functional.cross_entropy((h @ model.head.t()).flatten(0, 1), target.flatten())
        loss.backward()
        results.append((loss.item(), {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}))
    assert abs(results[0][0] - results[1][0]) <= 1e-5 * abs(results[1][0])
    assert results[0][1].keys() == results[1][1].keys()
    for n, g in results[0][1].items():
        want = results[1][1][n]
        assert (g - want).abs().max() <= 2e-4 * want.abs().max(), n


@pytest.mark.parametrize("bits", [8, 32])
def test_the_loss_falls(example, bits):
    """From log(31) on the uniform start; the data's own entropy is about 0.3."""
    losses = example.train(steps=60, vocab=31, width=48, rows=64, length=16, state_bits=bits, quiet=True)
    assert all(np.isfinite(losses))
    assert np.mean(losses[:3]) > 2.5 and np.mean(losses[-5:]) < 0.6 * np.mean(losses[:3]), (losses[:3], losses[-5:])
