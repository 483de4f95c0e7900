"""orthogonalize(), its gradient and muon() at the ends of the types' ranges, where a norm leaves a float's, in every class of sizes."""

import pytest
import torch

from tests import _newton_schulz as N
from tests.test_gpu_orthogonalize import data, gs

pytestmark = pytest.mark.gpu

# thin (a thread a matrix, a few lanes a matrix), one block, a cluster, tiles
SHAPES = [(70, 15, 3), (3, 4, 60), (2, 3, 110), (2, 40, 24), (1, 77, 1000), (1, 200, 136), (1, 5, 20000)]
TOP = 3e38  # the largest entry; 3.4e38 is the largest float


def scaled(shape, dtype, seed, top):
    x = data(shape, torch.float32, seed, 1.0)
    return (x / x.abs().amax((-2, -1), keepdim=True) * top).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_norm_above_the_largest_float(shape, dtype):
    x = scaled(shape, dtype, 300, TOP)
    assert (x.double().flatten(-2).norm(dim=-1) > 3.5e38).all()
    y = gs().orthogonalize(x.cuda()).cpu()
    assert N.distance(y, N.newton_schulz(x)) <= N.tolerance(x, 5, N.QUINTIC)


@pytest.mark.parametrize("shape", SHAPES)
def test_subnormal_matrix(shape):
    """Entries of 1e-39, which are multiples of 2^-149 and exact in 64 bits as they are in 32."""
    x = scaled(shape, torch.float32, 301, 1e-39)
    y = gs().orthogonalize(x.cuda(), eps=1e-44).cpu()
    eps = float(torch.tensor(1e-44, dtype=torch.float32))
    assert N.distance(y, N.newton_schulz(x, eps=eps)) <= N.tolerance(x, 5, N.QUINTIC, eps)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("top_x,top_v", [(TOP, 1e30), (1e37, 1e35), (1.0, 1e-34), (1e-32, 1e-34), (1e-20, 1e-37)])
def test_gradient_of_far_scales(shape, top_x, top_v):
    """The gradient goes with |v| / |x|. Thin matrices keep G in 32 bits, so v times the slope 485 stays below 3.4e38 here, and
    below 1e-30 they are let off by their subnormals' steps."""
    x, v = scaled(shape, torch.float32, 302, top_x), scaled(shape, torch.float32, 303, top_v)
    xg = x.cuda().requires_grad_(True)
    (got,) = torch.autograd.grad(gs().orthogonalize(xg, eps=1e-37), xg, v.cuda())
    # the same gradient of x and v of middle scales, by powers of two: what is compared stays exact
    sx, sv = (2.0 ** round(float(torch.log2(torch.tensor(t, dtype=torch.float64)))) for t in (top_x, top_v))
    xm, vm = (x.double() / sx), (v.double() / sv)
    exact = N.gradient(xm, vm, 5, N.QUINTIC, 1e-37)
    gm = got.cpu().double() * sx / sv
    tol = N.gradient_tolerance(xm.float(), vm.float(), 5, N.QUINTIC, 1e-37) * exact.norm() + N.projected_away(xm, vm, 5, N.QUINTIC, 1e-37)
    # a result below 2^-126 has a step of 2^-149
    step = 2.0**-150 * sx / sv * got.numel() ** 0.5
    assert float((gm - exact).norm()) <= float(tol) + step


def test_gradient_with_v_above_the_largest_norm():
    for shape in ((2, 40, 24), (1, 200, 136)):
        x, v = scaled(shape, torch.float32, 304, 1e4), scaled(shape, torch.float32, 305, TOP)
        xg = x.cuda().requires_grad_(True)
        (got,) = torch.autograd.grad(gs().orthogonalize(xg), xg, v.cuda())
        exact = N.gradient(x, v.double() * 2.0**-100, 5, N.QUINTIC)
        off = (got.cpu().double() * 2.0**-100 - exact).norm()
        small = v.double() * 2.0**-100
        assert off <= N.gradient_tolerance(x, small.float(), 5, N.QUINTIC) * exact.norm() + N.projected_away(x, small, 5, N.QUINTIC)


@pytest.mark.parametrize("shape", SHAPES)
def test_muon_with_norm_above_the_largest_float(shape):
    p, g = data(shape, torch.float32, 306, 0.02), scaled(shape, torch.float32, 307, TOP)
    tp, tm = p.cuda(), torch.zeros(shape, device="cuda")
    gs().muon(tp, g.cuda(), tm, None, 0.1, 0.9)
    # u is 0.19 of g, with roundings of its own that tolerance() counts as carried
    want = p.double() - 0.1 * N.newton_schulz(0.19 * g.double())
    allowed = 0.1 * N.tolerance(g, 5, N.QUINTIC) * N.newton_schulz(g).norm() + 4 * 2.0**-24 * want.norm()
    assert (tp.cpu().double() - want).norm() <= allowed


@pytest.mark.parametrize("length", [100_000, 8_000_000])
def test_square_of_a_long_row(length):
    """A = |x0|^2 = 1, a sum of squares that a truncating adder falls short of. With p = -15 s + 16 s^3 the result is x0, 16 times
    A's error off in length. bfloat16 operands have 11 bits here: their roundings, of 128 mantissas, leave the mean of
    squares 2 * 2^-12 / sqrt(128) off, 16 of which are 7e-4; and bfloat16 results scatter by 2^-9, which the mean forgets."""
    x = data((1, length), torch.bfloat16, 310, 1.0)
    y = gs().orthogonalize(x.cuda(), steps=1, coefficients=(-15.0, 16.0, 0.0)).cpu().double()
    x0 = x.double() / x.double().norm()
    assert abs(float((y * x0).sum()) - 1) < 2e-3
