"""Newton-Schulz orthogonalisation and the Muon step in 64 bits, for the tests, and how far rounding may
take a kernel from them."""

import torch

QUINTIC = (3.4445, -4.7750, 2.0315)
CUBIC = (1.5, -0.5, 0.0)
# relative to the value, a rounding is off by half a step at most
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def triples(coefficients, steps):
    return list(coefficients) if isinstance(coefficients[0], (tuple, list)) else [coefficients] * steps


def newton_schulz(x, steps=5, coefficients=QUINTIC, eps=1e-7, products=0.0, carried=0.0, gen=None):
    """x [..., M, N] in 64 bits. `products` / `carried`: the operands of the matrix products, and the X that goes from step to
    step, are off by so much of their value, at random: a model of a kernel's roundings (the diagonals
    of A and B, which the kernels keep in 32 bits, only by `carried`)."""
    x = x.double()
    if x.shape[-2] > x.shape[-1]:
        return newton_schulz(x.mT, steps, coefficients, eps, products, carried, gen).mT

    def off(t, by):
        if not by:
            return t
        return t * (1 + by * (2 * torch.rand(t.shape, generator=gen, dtype=torch.float64) - 1).to(t.device))

    def off_diagonal(t):
        if not products:
            return t
        d = torch.diag_embed(t.diagonal(dim1=-2, dim2=-1))
        return off(d, carried) + off(t - d, products)

    x = off(x / torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True).clamp_min(eps), carried)
    for a, b, c in triples(coefficients, steps):
        r = off(x, products)
        g = off_diagonal(r @ r.mT)
        x = off(a * x + off_diagonal(b * g + c * (g @ g)) @ r, carried)
    return x


def rounding(dtype, rows, cols):
    """(products, carried) of a kernel: bfloat16 matrices with a side above 128 are multiplied with 11 significand bits, all others with
    22; what is carried has 22. Each is doubled for the 32-bit sums beside it."""
    half = dtype == torch.bfloat16 and max(rows, cols) > 128
    return (2.0**-11 if half else 2.0**-21), 2.0**-21


def distance(a, b):
    """2-norm of the difference over that of b, over the whole tensor."""
    a, b = a.double(), b.double()
    n = b.norm()
    return float((a - b).norm() / n) if n > 0 else float((a - b).norm())


def tolerance(x, steps, coefficients, eps=1e-7):
    """What the model's roundings do to the result, eight times over (they are one draw, and a kernel's
    need not be random), and the rounding of the result."""
    gen = torch.Generator().manual_seed(3)
    products, carried = rounding(x.dtype, *x.shape[-2:])
    exact = newton_schulz(x, steps, coefficients, eps)
    return 8 * distance(newton_schulz(x, steps, coefficients, eps, products, carried, gen), exact) + HALF_STEP[x.dtype]


def gradient(x, v, steps, coefficients, eps=1e-7, **model):
    x = x.detach().double().requires_grad_(True)
    return torch.autograd.grad(newton_schulz(x, steps, coefficients, eps, **model), x, v.double())[0]


def gradient_tolerance(x, v, steps, coefficients, eps=1e-7):
    """The backward multiplies all types with 22 bits. Its own products round as the steps' do, so the
    factor is twice the forward's."""
    gen = torch.Generator().manual_seed(4)
    exact = gradient(x, v, steps, coefficients, eps)
    noisy = gradient(x, v, steps, coefficients, eps, products=2.0**-21, carried=2.0**-21, gen=gen)
    return 16 * distance(noisy, exact) + HALF_STEP[x.dtype]


def projected_away(x, v, steps, coefficients, eps=1e-7):
    """An absolute allowance for the gradient: dX0 - X0 <dX0, X0> cancels the part along X0 (all of it for a
    1 x 1 matrix), so roundings count relative to dX0 / |x|: 32 of 2^-24, a few for each step."""
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt().clamp_min(eps)
    x0 = (x.double() / norm).requires_grad_(True)
    y = x0
    for t in triples(coefficients, steps):
        y = _step(y, *t)
    return float(32 * 2.0**-24 * (torch.autograd.grad(y, x0, v.double())[0] / norm).norm())


def _step(x, a, b, c):
    g = x @ x.mT
    return a * x + (b * g + c * (g @ g)) @ x
