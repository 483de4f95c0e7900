"""The state that orthogonalize() keeps for its backward pass."""

import pytest
import torch

from tests import _newton_schulz as N
from tests.test_gpu_orthogonalize import data, gs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(1, 300, 200), (2, 129, 140)])
def test_state_of_a_forward_whose_wait_ran_out_gives_nan(shape):
    """The state's first word says so; the gradient must not look like one."""
    x, v = data(shape, torch.float32, 400).cuda().requires_grad_(True), data(shape, torch.float32, 401, 1.0).cuda()
    y = gs().orthogonalize(x)
    kept = y.grad_fn.saved_tensors[1].data
    assert kept[:4].tolist() == [0, 0, 0, 0]
    (first,) = torch.autograd.grad(y, x, v, retain_graph=True)
    assert torch.isfinite(first).all()
    kept[0] = 1
    assert torch.isnan(torch.autograd.grad(y, x, v, retain_graph=True)[0]).all()
    kept[0] = 0  # the mark is read, not reset
    assert torch.equal(torch.autograd.grad(y, x, v)[0], first)
