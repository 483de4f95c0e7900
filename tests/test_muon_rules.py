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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("momentum_dtype", [None, torch.float32])
def test_checkpoint_keeps_the_momentum(plain, dtype, momentum_dtype):
    """A saved and loaded state has the buffers' type and every bit of them, also through a file's copy."""
    import copy

    gen = torch.Generator().manual_seed(2)
    args = dict(lr=0.01, momentum_dtype=momentum_dtype)
    ps = [torch.nn.Parameter(torch.randn(6, 5, generator=gen).to(dtype)) for _ in range(3)]
    opt = gsplat_b200.Muon([dict(params=ps[:2]), dict(params=ps[2:], lr=0.5)], **args)
    for p in ps[:2]:
        p.grad = torch.randn(6, 5, generator=gen).to(dtype)
    opt.step()
    want = [opt.state[p]["momentum_buffer"] for p in ps[:2]]
    assert all(w.dtype == (momentum_dtype or dtype) for w in want)
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    other = gsplat_b200.Muon([dict(params=qs[:2]), dict(params=qs[2:])], **args)
    other.register_load_state_dict_pre_hook(lambda _, state: copy.deepcopy(state))  # a user's hook may replace the state
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    for q, w in zip(qs, want):
        got = other.state[q]["momentum_buffer"]
        assert got.dtype == w.dtype and torch.equal(got, w) and got.data_ptr() != w.data_ptr()
    assert "momentum_buffer" not in other.state[qs[2]] and other.param_groups[1]["lr"] == 0.5
    for p, q in zip(ps, qs):
        p.grad = torch.randn(6, 5, generator=gen).to(dtype)
        q.grad = p.grad.clone()
    opt.step(), other.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))


def test_state_of_torch_muon_is_taken(plain):
    ps = [torch.nn.Parameter(torch.ones(4, 6, dtype=torch.bfloat16)) for _ in range(2)]
    theirs = torch.optim.Muon(ps, lr=0.3)
    ps[0].grad = torch.ones(4, 6, dtype=torch.bfloat16)
    theirs.step()
    opt = gsplat_b200.Muon([torch.nn.Parameter(p.detach().clone()) for p in ps], momentum_dtype=torch.float32)
    opt.load_state_dict(theirs.state_dict())
    a, b = opt.param_groups[0]["params"]
    assert opt.param_groups[0]["lr"] == 0.3 and opt.state[a]["momentum_buffer"].dtype == torch.float32
    assert torch.equal(opt.state[a]["momentum_buffer"], theirs.state[ps[0]]["momentum_buffer"].float())
    b.grad = torch.ones(4, 6, dtype=torch.bfloat16)
    opt.step()
    assert opt.state[b]["momentum_buffer"].dtype == torch.float32


def test_step_takes_a_closure(plain):
    """As torch's optimizers do: called with gradients on, before the step, its value returned."""
    gen = torch.Generator().manual_seed(3)
    w = torch.randn(6, 5, generator=gen)
    ours, theirs = (torch.nn.Parameter(w.clone()) for _ in range(2))
    opt = gsplat_b200.Muon([ours], lr=0.1)
    other = gsplat_b200.Muon([theirs], lr=0.1)

    def closure():
        opt.zero_grad()
        loss = (ours * ours).sum()
        loss.backward()
        return loss

    (theirs * theirs).sum().backward()
    other.step()
    assert float(opt.step(closure)) == pytest.approx(float((w * w).sum()), rel=1e-6)
    assert torch.equal(ours, theirs) and not torch.equal(ours, w)
    assert float(opt.step(closure=closure)) < float((w * w).sum())
    assert opt.step() is None
    with pytest.raises(TypeError):
        opt.step(closure, closure)


def test_unsuitable_parameters_are_refused_before_the_first_step():
    half, full = torch.nn.Parameter(torch.ones(4, 4, dtype=torch.bfloat16)), torch.nn.Parameter(torch.ones(4, 4))
    for p, dtype in ((half, torch.float16), (full, torch.bfloat16), (full, torch.float64)):
        with pytest.raises(TypeError, match="momentum_dtype"):
            gsplat_b200.Muon([p], momentum_dtype=dtype)
    for p, dtype in ((half, torch.bfloat16), (half, torch.float32), (half, None), (full, torch.float32)):
        gsplat_b200.Muon([p], momentum_dtype=dtype)
    opt = gsplat_b200.Muon([full])
    for bad in (dict(params=[torch.nn.Parameter(torch.ones(4))]), dict(params=[half], momentum_dtype=torch.float16)):
        with pytest.raises((TypeError, ValueError)):
            opt.add_param_group(bad)
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[half], momentum_dtype=torch.float32))


def test_unsuitable_mask_leaves_all_groups_as_they_were(plain):
    rows, plain_matrix = torch.nn.Parameter(torch.ones(5, 4, 3)), torch.nn.Parameter(torch.ones(5, 4))
    for other in (plain_matrix, torch.nn.Parameter(torch.ones(6, 4, 3))):
        opt = gsplat_b200.Muon([dict(params=[rows]), dict(params=[other])])
        rows.grad, other.grad = torch.ones(5, 4, 3), torch.ones_like(other)
        with pytest.raises(ValueError, match="does not mask"):
            opt.step(torch.ones(5, dtype=torch.bool))
        assert (rows == 1).all() and not opt.state
    other.grad = None  # nothing to step there
    opt.step(torch.ones(5, dtype=torch.bool))
    assert (rows != 1).any()


def test_checkpoint_of_other_parameter_types(plain):
    """Buffers go to the new parameter's type where the saved momentum_dtype does not suit it, as torch casts them."""
    half = torch.nn.Parameter(torch.ones(4, 6, dtype=torch.bfloat16))
    opt = gsplat_b200.Muon([half], momentum_dtype=torch.bfloat16)
    half.grad = torch.ones(4, 6, dtype=torch.bfloat16)
    opt.step()
    full, fresh = torch.nn.Parameter(torch.ones(4, 6)), torch.nn.Parameter(torch.ones(4, 6))
    other = gsplat_b200.Muon([full])
    other.load_state_dict(opt.state_dict())
    assert other.state[full]["momentum_buffer"].dtype == torch.float32
    assert torch.equal(other.state[full]["momentum_buffer"], opt.state[half]["momentum_buffer"].float())
    other.param_groups[0]["params"].append(fresh)
    full.grad, fresh.grad = torch.ones(4, 6), torch.ones(4, 6)
    other.step()
    assert other.state[fresh]["momentum_buffer"].dtype == torch.float32
