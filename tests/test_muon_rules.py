"""CPU checks of the Muon class's rules against torch.optim.Muon, with the step itself in plain 64-bit form."""

import pytest
import torch

import gsplat_b200
from gsplat_b200.optimizers import muon as muon_module
from tests import _newton_schulz as N


def plain_muon(params, grads, buffers, valid, lr, momentum, weight_decay=0.0, nesterov=True, steps=5,
               coefficients=N.QUINTIC, eps=1e-7, update_scale=1.0):
    """muon() as it documents itself."""
    scales = update_scale if isinstance(update_scale, list) else [update_scale] * len(params)
    for p, g, m, scale in zip(params, grads, buffers, scales):
        m += (1 - momentum) * (g - m)
        u = g + momentum * (m - g) if nesterov else m
        p.copy_(p * (1 - lr * weight_decay) - lr * scale * N.newton_schulz(u, steps, coefficients, eps))


@pytest.fixture
def plain(monkeypatch):
    monkeypatch.setattr(muon_module, "muon", plain_muon)


@pytest.mark.parametrize("rule", [None, "original", "match_rms_adamw"])
@pytest.mark.parametrize("shape", [(4096, 8), (15, 3), (8, 64), (32, 32)])
def test_weight_decay_goes_by_the_learning_rate_alone(plain, shape, rule):
    """With zero gradients a step only decays: by 1 - lr weight_decay, whatever the shape, as torch's does."""
    ours, theirs = (torch.nn.Parameter(torch.ones(shape)) for _ in range(2))
    ours.grad, theirs.grad = torch.zeros(shape), torch.zeros(shape)
    args = dict(lr=0.02, weight_decay=0.1, adjust_lr_fn=rule)
    gsplat_b200.Muon([ours], **args).step()
    torch.optim.Muon([theirs], **args).step()
    # both round 1 - 0.002 to 32 bits, and the product once
    assert (ours - theirs).abs().max() <= 2 * 2.0**-24
    assert (ours.double() - 0.998).abs().max() <= 2 * 2.0**-24


@pytest.mark.parametrize("rule", [None, "match_rms_adamw"])
@pytest.mark.parametrize("shape", [(60, 4), (15, 3), (8, 20)])
def test_update_is_scaled_by_the_shape(plain, shape, rule):
    """The update's own size, without a decay: torch takes its products in bfloat16, whose roundings (2^-8 of values up to
    1.2, in 15 products) leave it within a fifth; the factors here are 1, 1.8, 2.2, 3.9 and 0.8 to 1.5."""
    gen = torch.Generator().manual_seed(1)
    g = torch.randn(shape, generator=gen)
    ours, theirs = (torch.nn.Parameter(torch.zeros(shape)) for _ in range(2))
    ours.grad, theirs.grad = g.clone(), g.clone()
    args = dict(lr=0.02, weight_decay=0.0, adjust_lr_fn=rule)
    gsplat_b200.Muon([ours], **args).step()
    torch.optim.Muon([theirs], **args).step()
    assert N.distance(ours.detach(), theirs.detach()) < 0.2
