"""The Muon class and muon()'s arguments on the GPU against 64-bit implementations."""

import copy
import math

import pytest
import torch

from tests import _newton_schulz as N
from tests.test_gpu_orthogonalize import data, gs, step64

pytestmark = pytest.mark.gpu


def off_by(got, p, g, m, lr, scale, mu, wd):
    """(distance from the 64-bit step, what roundings allow): the update to 485 (the steps' largest slope) 22-bit roundings,
    the parameter to three 32-bit operations. step64 gives the update (no decay, lr 1, from a zero parameter)."""
    o = -step64(torch.zeros_like(p), g, m, None, 1.0, mu, 0.0, True)[0]
    want = p.double() * (1 - lr * wd) - lr * scale * o
    return float((got.cpu().double() - want).norm()), float(485 * 2.0**-21 * lr * scale * o.norm() + 4 * 2.0**-24 * p.double().norm())


@pytest.mark.parametrize("rule", [None, "match_rms_adamw"])
def test_weight_decay_goes_by_the_learning_rate_alone(rule):
    shapes = [(400, 8), (15, 3), (64, 300), (300, 130)]
    ps = [torch.nn.Parameter(data(s, torch.float32, 200 + i, 1.0).cuda()) for i, s in enumerate(shapes)]
    before = [p.detach().cpu().clone() for p in ps]
    for i, p in enumerate(ps):
        p.grad = data(tuple(p.shape), torch.float32, 210 + i).cuda()
    gs().Muon(ps, lr=0.02, weight_decay=0.1, momentum=0.9, adjust_lr_fn=rule).step()
    for p, b in zip(ps, before):
        scale = 0.2 * math.sqrt(max(p.shape)) if rule else math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
        off, allowed = off_by(p.detach(), b, p.grad.cpu(), torch.zeros_like(b), 0.02, scale, 0.9, 0.1)
        assert off <= allowed  # a decay by lr times the factor is at least 0.0002 of |p| off, 20 times that


def test_update_scale_of_one_tensor_and_of_a_list():
    shapes = [(9, 15, 3), (40, 30), (150, 140)]
    ps, grads, ms = ([data(s, torch.float32, 220 + 3 * i + j, 0.5) for i, s in enumerate(shapes)] for j in range(3))
    tp, tm = [p.cuda() for p in ps], [m.cuda() for m in ms]
    gs().muon(tp, [g.cuda() for g in grads], tm, None, [0.1, 0.2, 0.3], 0.9, 0.5, update_scale=[2.0, 0.5, 0.0])
    for p, g, m, got, lr, scale in zip(ps, grads, ms, tp, (0.1, 0.2, 0.3), (2.0, 0.5, 0.0)):
        off, allowed = off_by(got, p, g, m, lr, scale, 0.9, 0.5)
        assert off <= allowed
    one, tm = ps[1].cuda(), ms[1].cuda()
    gs().muon(one, grads[1].cuda(), tm, None, 0.2, 0.9, 0.5, update_scale=0.5)
    assert torch.equal(one, tp[1])
    with pytest.raises(ValueError, match="same length"):
        gs().muon(tp, [g.cuda() for g in grads], [m.cuda() for m in ms], None, 0.1, 0.9, update_scale=[1.0])


def test_visibility_and_checkpoint():
    """Per-splat SH bands under a visibility mask, with the momentum in 32 bits, and a checkpoint of it."""
    sh = torch.nn.Parameter(data((30, 15, 3), torch.bfloat16, 60, 1.0).cuda())
    opt = gs().Muon([sh], lr=0.1, momentum_dtype=torch.float32)
    before = sh.detach().clone()
    sh.grad = data((30, 15, 3), torch.bfloat16, 61).cuda()
    vis = torch.arange(30, device="cuda") % 2 == 0
    opt.step(vis)
    assert torch.equal(sh.detach()[~vis], before[~vis]) and (sh.detach()[vis] != before[vis]).flatten(1).any(1).all()
    buffer = opt.state[sh]["momentum_buffer"]
    assert buffer.dtype == torch.float32 and (buffer[~vis] == 0).all()
    q = torch.nn.Parameter(sh.detach().clone())
    other = gs().Muon([q], lr=0.5, momentum_dtype=torch.float32)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert torch.equal(other.state[q]["momentum_buffer"], buffer)
    q.grad = sh.grad.clone()
    opt.step(vis)
    other.step(vis)
    assert torch.equal(q.detach(), sh.detach()) and torch.equal(other.state[q]["momentum_buffer"], buffer)


@pytest.mark.parametrize("shape", [(300, 15, 3), (2, 4, 60), (40, 30), (200, 140)])
def test_momentum_near_one(shape):
    """1 - 0.9999 to 32 bits: from a buffer of zeros m = (1 - momentum) g, in three roundings."""
    p, g = data(shape, torch.float32, 230, 0.1).cuda(), data(shape, torch.float32, 231, 1.0).cuda()
    m = torch.zeros_like(p)
    gs().muon(p, g, m, None, 0.1, 0.9999)
    want = (1 - 0.9999) * g.double()
    assert ((m.double() - want).abs() <= 3 * 2.0**-24 * want.abs()).all()
