"""CPU checks of orthogonalize() with the launch replaced: derivatives that it does not have, and its coefficients."""

import pytest
import torch

import gsplat_b200
from gsplat_b200.cuda import _wrapper


@pytest.fixture
def launches(monkeypatch):
    """The coefficients of each launch; the result is twice the input."""
    seen = []

    def fwd(x, steps, coefficients, eps, keep=False):
        seen.append(list(coefficients))
        return (2 * x.detach(), None) if keep else 2 * x.detach()

    monkeypatch.setattr(_wrapper, "_orthogonalize_fwd", fwd)
    return seen


def test_forward_mode_is_refused(launches):
    x = torch.randn(3, 3)
    with torch.autograd.forward_ad.dual_level():
        for base in (x, x.clone().requires_grad_(True)):
            dual = torch.autograd.forward_ad.make_dual(base, torch.ones_like(x))
            with pytest.raises(NotImplementedError, match="forward"):
                gsplat_b200.orthogonalize(dual)
        gsplat_b200.orthogonalize(x)  # has no tangent
    with pytest.raises(NotImplementedError):
        torch.func.jvp(gsplat_b200.orthogonalize, (x,), (torch.ones_like(x),))
    assert len(launches) == 1


@pytest.mark.parametrize("nested", [False, True])
def test_coefficients_are_read_at_each_call(launches, nested):
    """Of tensors that change in place (an annealed schedule), as of new numbers."""
    triple = [torch.tensor(1.5), torch.tensor(-0.5), torch.tensor(0.0)]
    coefficients = [triple, (3.0, -2.0, 0.0)] if nested else triple
    rest = [3.0, -2.0, 0.0] if nested else []
    x = torch.randn(3, 3)
    gsplat_b200.orthogonalize(x, len(rest) // 3 + 1, coefficients)
    triple[0].fill_(2.0)
    gsplat_b200.orthogonalize(x, len(rest) // 3 + 1, coefficients)
    gsplat_b200.orthogonalize(x, 1, torch.tensor([1.25, -0.25, 0.0]))
    gsplat_b200.orthogonalize(x, 2, torch.tensor([[1.25, -0.25, 0.0], [1.0, 0.0, 0.5]]))
    assert launches == [[1.5, -0.5, 0.0] + rest, [2.0, -0.5, 0.0] + rest, [1.25, -0.25, 0.0], [1.25, -0.25, 0.0, 1.0, 0.0, 0.5]]
