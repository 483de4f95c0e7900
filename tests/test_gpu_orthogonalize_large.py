"""The tiled products at sizes that take every kind of tile (tests/test_orthogonalize_tiles.py holds which), batches that are taken
in pieces and a state too large to keep, against 64-bit implementations on the same GPU."""

import math

import pytest
import torch

from tests import _newton_schulz as N
from tests._tiles import TILES
from tests.test_gpu_orthogonalize import data, gs, step64

pytestmark = pytest.mark.gpu

PIECES = (3700, 130, 150)  # scratch of 1.1 GiB, where 1 is taken at a time


def made(shape, dtype, seed, scale=1e-4):
    """As data(), on the GPU."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=gen, device="cuda")
    r = max(1, min(shape[-2:]) // 8)
    x += (torch.randn(*shape[:-1], r, generator=gen, device="cuda") @ torch.randn(*shape[:-2], r, shape[-1], generator=gen, device="cuda")) / r**0.5
    return (x * scale).to(dtype)


def per_matrix(a, b):
    """The largest distance of a matrix, so that a wrong one among many is seen."""
    a, b = a.double().flatten(-2), b.double().flatten(-2)
    return float(((a - b).norm(dim=-1) / b.norm(dim=-1)).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("shape", TILES)
def test_orthogonalize(shape, turned, dtype):
    x = made((shape[0], shape[2], shape[1]) if turned else shape, dtype, 500)
    y = gs().orthogonalize(x)
    # the model's distance is of the whole batch; its matrices are alike, and one is off by twice the mean at most
    assert per_matrix(y, N.newton_schulz(x)) <= 2 * N.tolerance(x, 5, N.QUINTIC)


def check_gradient(x, v, got):
    exact = N.gradient(x, v, 5, N.QUINTIC)
    off = (got.double() - exact).norm()
    assert off <= N.gradient_tolerance(x, v, 5, N.QUINTIC) * exact.norm() + N.projected_away(x, v, 5, N.QUINTIC)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", TILES)
def test_gradient(shape, dtype):
    if shape[1] % 2 == 0 and dtype == torch.bfloat16:  # the other orientation for half of them
        shape = (shape[0], shape[2], shape[1])
    x, v = made(shape, dtype, 501).requires_grad_(True), made(shape, dtype, 502, 1.0)
    y = gs().orthogonalize(x)
    # with a state to keep, 16-bit matrices are multiplied with 22 bits too
    assert per_matrix(y.detach(), N.newton_schulz(x.detach())) <= 2 * N.tolerance(x.detach().float(), 5, N.QUINTIC) + 2 * N.HALF_STEP[dtype]
    (got,) = torch.autograd.grad(y, x, v)
    check_gradient(x.detach(), v, got)


@pytest.mark.parametrize("dtype,state", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                         (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
def test_muon_of_large_matrices_under_a_mask(dtype, state):
    """Both orientations together, with hidden matrices whose gradient is NaN, at 256-wide and 128-wide tiles and odd sizes."""
    shapes = [(3, 1500, 1700), (3, 1700, 1500), (3, 1100, 2300), (3, 20, 300, 520), (3, 20, 520, 300), (3, 129, 131)]
    ps = [made(s, dtype, 510 + i, 0.02) for i, s in enumerate(shapes)]
    ms = [made(s, state, 520 + i, 1e-2) for i, s in enumerate(shapes)]
    grads = [made(s, dtype, 530 + i, 1e-2) for i, s in enumerate(shapes)]
    for g in grads:
        g[1] = math.nan
    valid = torch.tensor([True, False, True], device="cuda")
    tp, tm = [p.clone() for p in ps], [m.clone() for m in ms]
    gs().muon(tp, grads, tm, valid, 0.03, 0.95, 0.1)
    for p, g, m, got_p, got_m in zip(ps, grads, ms, tp, tm):
        assert torch.equal(got_p[1], p[1]) and torch.equal(got_m[1], m[1])
        p, g, m, got_p, got_m = (t[valid] for t in (p, g, m, got_p, got_m))
        q, n = step64(p, g, m, None, 0.03, 0.95, 0.1, True)
        assert per_matrix(got_m, n) <= N.HALF_STEP[state] + 4 * 2.0**-24
        products, carried = N.rounding(dtype, *p.shape[-2:])
        gen = torch.Generator().manual_seed(5)
        model = step64(p, g, m, None, 0.03, 0.95, 0.1, True, products=products, carried=carried, gen=gen)[0]
        assert per_matrix(got_p, q) <= 16 * N.distance(model, q) + 2 * N.HALF_STEP[dtype] + 4 * 2.0**-24


def test_batch_taken_in_pieces():
    from gsplat_b200.cuda import _backend

    L = _backend.lib()
    assert L.gsb_orthogonalize_scratch_bytes(*PIECES, 0, 5, 0, 0) == L.gsb_orthogonalize_scratch_bytes(2 * PIECES[0], *PIECES[1:], 0, 5, 0, 0)
    x = made(PIECES, torch.float32, 540)
    x[3600] = math.nan
    y = gs().orthogonalize(x)
    assert torch.isnan(y[3600]).all()
    x[3600], y[3600] = x[0], y[0]
    assert per_matrix(y, N.newton_schulz(x)) <= 2 * N.tolerance(x[:100].cpu(), 5, N.QUINTIC)


def test_gradient_of_a_batch_taken_in_pieces():
    """Its state is not kept either, and taken again piece by piece."""
    from gsplat_b200.cuda import _backend

    assert _backend.lib().gsb_orthogonalize_kept_bytes(*PIECES, 5) == 0
    x, v = made(PIECES, torch.float32, 541).requires_grad_(True), made(PIECES, torch.float32, 542, 1.0)
    (got,) = torch.autograd.grad(gs().orthogonalize(x), x, v)
    at = [0, 1, 700, 760, 1500, 2222, 3500, 3699]
    xs, vs = x.detach(), v
    for i in range(0, PIECES[0], 500):
        exact = N.gradient(xs[i : i + 500], vs[i : i + 500], 5, N.QUINTIC)
        # a first look at all of them; the tolerance itself at some
        assert per_matrix(got[i : i + 500], exact) < 1e-3
    check_gradient(xs[at], vs[at], got[at])


def test_gradient_without_state_at_its_size():
    """One matrix whose state would be above 1 GiB with the scratch."""
    from gsplat_b200.cuda import _backend

    shape = (1, 3900, 4200)
    assert _backend.lib().gsb_orthogonalize_kept_bytes(*shape, 5) == 0
    x, v = made(shape, torch.float32, 543).requires_grad_(True), made(shape, torch.float32, 544, 1.0)
    y = gs().orthogonalize(x)
    assert y.grad_fn.saved_tensors[1] is None
    (got,) = torch.autograd.grad(y, x, v)
    check_gradient(x.detach(), v, got)


def test_muon_step_taken_in_pieces():
    """A piece ends inside a tensor, and the mask goes by the place in the tensor."""
    n = PIECES[0] // 4
    shapes = [(n, 130, 150), (n, 2, 150, 130), (n, 130, 150)]
    ps, grads, ms = ([made(s, torch.float32, 550 + 3 * i + j, 0.02) for i, s in enumerate(shapes)] for j in range(3))
    valid = torch.rand(n, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") < 0.7
    tp, tm = [p.clone() for p in ps], [m.clone() for m in ms]
    gs().muon(tp, grads, tm, valid, 0.1, 0.9, 0.1)
    for p, g, m, got_p, got_m in zip(ps, grads, ms, tp, tm):
        assert torch.equal(got_p[~valid], p[~valid]) and torch.equal(got_m[~valid], m[~valid])
        q, k = step64(p[valid], g[valid], m[valid], None, 0.1, 0.9, 0.1, True)
        assert per_matrix(got_m[valid], k) <= 5 * 2.0**-24
        # the update has a norm of about 11, lr 0.1 of it; the parameter's is about 3.5 and its rounding beside that
        tol = 2 * N.tolerance(g[:50].cpu(), 5, N.QUINTIC)
        assert per_matrix(got_p[valid], q) <= tol + 5 * 2.0**-24


def test_deep_products_of_bfloat16():
    """Short sides above 16384: every product of hi alone is read out on its way. The model's distance is taken of a smaller
    matrix of the same make; it does not grow with the side, whose roundings are independent."""
    shape, steps = (1, 16400, 16500), 2
    x = made(shape, torch.bfloat16, 560)
    want = N.newton_schulz(x, steps)
    tol = N.tolerance(made((1, 2000, 2100), torch.bfloat16, 561).cpu(), steps, N.QUINTIC)
    assert per_matrix(gs().orthogonalize(x, steps), want) <= 2 * tol
    p, m = torch.zeros_like(x), torch.zeros_like(x)
    gs().muon(p, x, m, None, 1.0, 0.0, nesterov=False, steps=steps)
    assert per_matrix(-p, want) <= 2 * tol
