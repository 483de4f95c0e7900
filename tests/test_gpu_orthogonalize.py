"""orthogonalize(), its gradient, muon() and the Muon optimizer against 64-bit implementations."""

import copy
import math

import pytest
import torch

from tests import _newton_schulz as N

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.bfloat16, torch.float16]
# both sides of every kernel's limits, odd sizes, tall and wide, one row, one column
MANY = [(8200, 1, 1), (9000, 3, 3), (8193, 15, 3), (8300, 2, 7), (8195, 4, 25), (8200, 32, 2), (8200, 4, 33), (8192, 16, 4)]
SHAPES = MANY + [(1, 1, 1), (3, 1, 7), (2, 7, 1), (1, 1, 300), (5, 2, 3), (70, 3, 3), (33, 15, 3), (9, 3, 16), (4, 4, 128),
          (2, 129, 4), (3, 5, 5), (2, 5, 131), (2, 64, 64), (1, 64, 35), (2, 100, 128), (1, 128, 128), (2, 128, 129),
          (1, 129, 127), (3, 16, 16), (2, 17, 1000), (2, 1000, 77), (1, 100, 700), (1, 128, 1024),
          (1, 1100, 128), (1, 5, 2300), (2, 48, 95), (1, 3, 20000), (1, 6000, 20), (1, 200, 4100), (2, 257, 65), (1, 300, 300), (1, 130, 517), (1, 513, 384)]


def gs():
    import gsplat_b200

    return gsplat_b200


def data(shape, dtype, seed=0, scale=1e-4):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen)
    r = max(1, min(shape[-2:]) // 8)
    x = x + torch.randn(*shape[:-1], r, generator=gen) @ torch.randn(*shape[:-2], r, shape[-1], generator=gen) / r**0.5
    return (x * scale).to(dtype)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(shape, dtype):
    x = data(shape, dtype)
    y = gs().orthogonalize(x.cuda())
    assert y.shape == x.shape and y.dtype == dtype
    assert N.distance(y.cpu(), N.newton_schulz(x)) <= N.tolerance(x, 5, N.QUINTIC)


@pytest.mark.parametrize("shape", [(6, 3, 3), (2, 30, 40), (1, 140, 150)])
@pytest.mark.parametrize("steps,coefficients", [(1, N.QUINTIC), (12, N.CUBIC), (32, N.CUBIC),
                                                (3, [(3.0, -3.2, 1.2), N.QUINTIC, N.CUBIC])])
def test_steps_and_coefficients(shape, steps, coefficients):
    x = data(shape, torch.float32, 1)
    y = gs().orthogonalize(x.cuda(), steps=steps, coefficients=coefficients).cpu()
    assert N.distance(y, N.newton_schulz(x, steps, coefficients)) <= N.tolerance(x, steps, coefficients)


def test_rotations_become_orthogonal():
    """The cubic on near-rotations converges quadratically: after 9 steps the result is orthogonal to 32-bit rounding."""
    x = torch.linalg.qr(torch.randn(500, 3, 3))[0] + 0.05 * torch.randn(500, 3, 3)
    y = gs().orthogonalize(x.cuda(), steps=9, coefficients=N.CUBIC).cpu().double()
    u, _, v = torch.linalg.svd(x.double())
    # singular values in 0.35 to 0.82 of the norm come to 1 within rounding; 9 steps of a 3-term sum
    assert (y - u @ v).abs().max() < 2.0**-24 * 9 * 9
    assert (y @ y.mT - torch.eye(3, dtype=torch.float64)).abs().max() < 2.0**-24 * 9 * 9


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", [(4, 3, 3), (2, 40, 24), (1, 200, 136)])
def test_extreme_scales_and_zero(shape, dtype):
    """The norm is divided out: tiny and huge inputs, a zero matrix, and one below eps."""
    for scale in (2.0**-12, 2.0**12) if dtype == torch.float16 else (1e-30, 1e30):
        eps = 1e-7 if dtype == torch.float16 else 1e-37
        x = data(shape, dtype, 2, scale)
        y = gs().orthogonalize(x.cuda(), eps=eps).cpu()
        assert N.distance(y, N.newton_schulz(x, eps=eps)) <= N.tolerance(x, 5, N.QUINTIC, eps)
    x = data(shape, dtype, 3)
    x[0] = 0
    y = gs().orthogonalize(x.cuda()).cpu()
    assert (y[0] == 0).all() and torch.isfinite(y.float()).all()
    x = data(shape, dtype, 4, 1e-3)
    y = gs().orthogonalize(x.cuda(), eps=1e3).cpu()
    exact = N.newton_schulz(x, eps=1e3)
    # far below eps each step is X <- a X. What is carried has an absolute step too, 2^-37 at a norm of 1 (485 = a^5
    # times), and a subnormal fp16 result one of 2^-24
    step = 485 * 2.0**-37 + (2.0**-25 if dtype == torch.float16 else 0.0)
    assert (y.double() - exact).norm() <= N.tolerance(x, 5, N.QUINTIC, 1e3) * exact.norm() + step * math.sqrt(x.numel())


@pytest.mark.parametrize("shape", [(3, 3, 4), (3, 20, 30), (2, 140, 150)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_non_finite_matrix_is_nan_and_alone(shape, bad):
    x = data(shape, torch.float32, 5)
    clean = gs().orthogonalize(x.cuda()).cpu()
    x[1, 1, 2] = bad
    y = gs().orthogonalize(x.cuda()).cpu()
    assert torch.isnan(y[1]).all()
    assert torch.equal(y[0], clean[0]) and torch.equal(y[2:], clean[2:])


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("shape", SHAPES)
def test_gradient(shape, dtype):
    x, v = data(shape, dtype, 6), data(shape, dtype, 7, 1.0)
    xg = x.cuda().requires_grad_(True)
    y = gs().orthogonalize(xg)
    (got,) = torch.autograd.grad(y, xg, v.cuda())
    assert got.dtype == dtype
    # entries are as large as 1 / |x|: fp16 overflows there, so it is compared where its own rounding is finite
    exact = N.gradient(x, v, 5, N.QUINTIC)
    finite = torch.isfinite(exact.to(dtype).float()) & torch.isfinite(got.cpu().float())
    if dtype != torch.float16:
        assert finite.all()
    off = (got.cpu().double() - exact)[finite].norm()
    assert off <= N.gradient_tolerance(x, v, 5, N.QUINTIC) * exact.norm() + N.projected_away(x, v, 5, N.QUINTIC)


@pytest.mark.parametrize("shape", [(3, 3, 3), (2, 12, 20), (1, 150, 140)])
@pytest.mark.parametrize("steps,coefficients", [(1, N.QUINTIC), (7, N.QUINTIC), (20, N.CUBIC)])
def test_gradient_steps(shape, steps, coefficients):
    x, v = data(shape, torch.float32, 8), data(shape, torch.float32, 9, 1.0)
    xg = x.cuda().requires_grad_(True)
    (got,) = torch.autograd.grad(gs().orthogonalize(xg, steps=steps, coefficients=coefficients), xg, v.cuda())
    exact = N.gradient(x, v, steps, coefficients)
    off = (got.cpu().double() - exact).norm()
    assert off <= N.gradient_tolerance(x, v, steps, coefficients) * exact.norm() + N.projected_away(x, v, steps, coefficients)


@pytest.mark.parametrize("shape", [(3, 20, 40), (2, 70, 500), (2, 150, 140)])
def test_gradient_without_kept_state(shape, monkeypatch):
    """Where the steps' state would be too large, the backward pass takes the steps again."""
    from gsplat_b200.cuda import _wrapper

    x, v = data(shape, torch.float32, 18), data(shape, torch.float32, 19, 1.0)
    xg = x.cuda().requires_grad_(True)
    monkeypatch.setattr(_wrapper, "_ortho_kept_bytes", lambda *a: 0)
    (got,) = torch.autograd.grad(gs().orthogonalize(xg), xg, v.cuda())
    exact = N.gradient(x, v, 5, N.QUINTIC)
    off = (got.cpu().double() - exact).norm()
    assert off <= N.gradient_tolerance(x, v, 5, N.QUINTIC) * exact.norm() + N.projected_away(x, v, 5, N.QUINTIC)


def test_gradient_twice_from_one_forward():
    """A retained graph: the kept state serves both passes."""
    for shape in ((5, 24, 40), (1, 300, 200)):
        x, v = data(shape, torch.float32, 90).cuda().requires_grad_(True), data(shape, torch.float32, 91, 1.0).cuda()
        y = gs().orthogonalize(x)
        first = torch.autograd.grad(y, x, v, retain_graph=True)[0]
        assert torch.equal(torch.autograd.grad(y, x, v)[0], first)


def test_gradient_against_differences():
    """A central difference of the kernel's own values along one direction: its error is the third derivative's h^2
    and the rounding 2^-22 / h of a sum of values of order 1."""
    x, v, d = (data((1, 24, 40), torch.float32, s, 1.0) for s in (10, 11, 12))
    f = lambda t: float((gs().orthogonalize(t.cuda()).cpu().double() * v.double()).sum())  # noqa: E731
    xg = x.cuda().requires_grad_(True)
    (g,) = torch.autograd.grad(gs().orthogonalize(xg), xg, v.cuda())
    slope = float((g.cpu().double() * d.double()).sum())
    h = 1e-3
    e = lambda t: float((N.newton_schulz(t) * v.double()).sum())  # noqa: E731
    truncation = abs((e(x.double() + h * d.double()) - e(x.double() - h * d.double())) / (2 * h) - slope)
    rounding = N.tolerance(x, 5, N.QUINTIC) * float(N.newton_schulz(x).norm() * v.double().norm()) / h
    assert abs((f(x + h * d) - f(x - h * d)) / (2 * h) - slope) <= 2 * truncation + 2 * rounding


def test_gradient_of_small_and_zero_matrices():
    for shape in ((3, 3, 3), (3, 10, 10), (3, 130, 140)):
        x, v = data(shape, torch.float32, 13), data(shape, torch.float32, 14, 1.0)
        x[0], v[1] = 0, 0
        xg = x.cuda().requires_grad_(True)
        (got,) = torch.autograd.grad(gs().orthogonalize(xg, eps=1e-3), xg, v.cuda())
        exact = N.gradient(x, v, 5, N.QUINTIC, 1e-3)
        assert (got[1] == 0).all()
        for b in range(3):
            one = x[b : b + 1], v[b : b + 1], 5, N.QUINTIC, 1e-3
            off = (got[b].cpu().double() - exact[b]).norm()
            assert off <= N.gradient_tolerance(*one) * exact[b].norm() + N.projected_away(*one)


def test_second_gradient_is_refused():
    x = data((2, 3, 3), torch.float32).cuda().requires_grad_(True)
    (g,) = torch.autograd.grad(gs().orthogonalize(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_batch_dimensions_strides_and_empty():
    x = data((4, 6, 5, 24), torch.float32, 15).cuda()
    y = gs().orthogonalize(x)
    assert torch.equal(y[1, 2], gs().orthogonalize(x[1, 2]))
    assert torch.equal(gs().orthogonalize(x.mT.contiguous().mT), y)
    assert torch.equal(gs().orthogonalize(x[::2, 1:4]), y[::2, 1:4])
    for shape in ((0, 3, 3), (2, 0, 5), (3, 5, 0), (0, 200, 200)):
        z = torch.empty(shape, device="cuda", requires_grad=True)
        y = gs().orthogonalize(z)
        assert y.shape == shape
        y.sum().backward()
        assert z.grad.shape == shape


def test_same_bits_each_time():
    for shape, dtype in (((50, 15, 3), torch.float32), ((2, 300, 200), torch.float32), ((1, 300, 700), torch.bfloat16)):
        x, v = data(shape, dtype, 16).cuda().requires_grad_(True), data(shape, dtype, 17, 1.0).cuda()
        first = gs().orthogonalize(x)
        grad = torch.autograd.grad(first, x, v)[0]
        for _ in range(3):
            y = gs().orthogonalize(x)
            assert torch.equal(y, first) and torch.equal(torch.autograd.grad(y, x, v)[0], grad)


# --- the step --------------------------------------------------------------------
def step64(p, g, m, valid, lr, mu, wd, nesterov, steps=5, coefficients=N.QUINTIC, **model):
    p, g, m0 = p.double(), g.double(), m.double()
    m = m0 + (1 - mu) * (g - m0)
    o = N.newton_schulz(g + mu * (m - g) if nesterov else m, steps, coefficients, **model)
    q = p * (1 - lr * wd) - lr * o
    if valid is not None:
        keep = valid.reshape([-1] + [1] * (p.dim() - 1))
        m, q = torch.where(keep, m, m0), torch.where(keep, q, p)
    return q, m


def check_step(p, g, m, got_p, got_m, valid, lr, mu, wd, nesterov):
    """The buffer to its type's rounding and three 32-bit operations; the parameter to that and lr times the
    orthogonalisation's tolerance."""
    q, n = step64(p, g, m, valid, lr, mu, wd, nesterov)
    assert N.distance(got_m, n) <= N.HALF_STEP[m.dtype] + 4 * 2.0**-24
    gen = torch.Generator().manual_seed(5)
    products, carried = N.rounding(p.dtype, *p.shape[-2:])
    model = step64(p, g, m, valid, lr, mu, wd, nesterov, products=products, carried=carried, gen=gen)[0]
    assert N.distance(got_p, q) <= 8 * N.distance(model, q) + N.HALF_STEP[p.dtype] + 4 * 2.0**-24
    if valid is not None:
        assert torch.equal(got_p[~valid], p[~valid]) and torch.equal(got_m[~valid], m[~valid])


@pytest.mark.parametrize("dtype,state", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                         (torch.bfloat16, torch.float32), (torch.float16, torch.float32),
                                         (torch.float16, torch.float16)])
@pytest.mark.parametrize("shape", [(8200, 15, 3), (2, 4100, 4, 9), (9001, 3, 30), (1, 1), (41, 3), (7, 15, 3), (3, 4, 20), (64, 35), (2, 3, 30, 40), (200, 140), (3, 150, 300)])
@pytest.mark.parametrize("nesterov", [True, False])
def test_muon(shape, dtype, state, nesterov):
    p, g, m = data(shape, dtype, 20, 0.02), data(shape, dtype, 21, 1e-2), data(shape, state, 22, 1e-2)
    tp, tg, tm = p.cuda(), g.cuda(), m.cuda()
    gs().muon(tp, tg, tm, None, 0.03, 0.95, 0.1, nesterov)
    assert torch.equal(tg.cpu(), g)
    check_step(p, g, m, tp.cpu(), tm.cpu(), None, 0.03, 0.95, 0.1, nesterov)


@pytest.mark.parametrize("shape", [(8300, 15, 3), (4200, 2, 3, 8), (67, 15, 3), (40, 2, 3, 8), (12, 20, 30), (5, 140, 150)])
def test_muon_valid(shape):
    p, g, m = (data(shape, torch.float32, s, 0.02) for s in (23, 24, 25))
    gen = torch.Generator().manual_seed(0)
    g[0] = math.nan  # hidden: not read
    for visible in (0.5, 0.0, 1.0):
        valid = torch.rand(shape[0], generator=gen) < visible
        valid[0] = False
        tp, tm = p.cuda(), m.cuda()
        gs().muon(tp, g.cuda(), tm, valid.cuda(), 0.1, 0.9, 0.0)
        assert torch.equal(tp.cpu()[~valid], p[~valid]) and torch.equal(tm.cpu()[~valid], m[~valid])
        if valid.any():
            check_step(p[valid], g[valid], m[valid], tp.cpu()[valid], tm.cpu()[valid], None, 0.1, 0.9, 0.0, True)


def test_muon_refusals():
    p, g, m = (torch.randn(6, 4, 5, device="cuda") for _ in range(3))
    ok = dict(momentum=0.9)
    with pytest.raises(ValueError, match="overlap"):
        gs().muon([p, p], [g, g], [m, m.clone()], None, 0.1, **ok)  # the same parameter twice
    with pytest.raises(ValueError, match="overlap"):
        gs().muon(p, p, m, None, 0.1, **ok)
    with pytest.raises(ValueError, match="overlap"):
        gs().muon([p[:4], p[2:]], [g[:4], g[2:]], [m[:4], m[:4].clone()], None, 0.1, **ok)
    gs().muon([p, p.clone()], [g, g], [m, m.clone()], None, 0.1, **ok)  # a gradient may serve two
    with pytest.raises(ValueError, match="alike"):
        gs().muon(p, g[:5], m, None, 0.1, **ok)
    with pytest.raises(TypeError):
        gs().muon(p, g.half(), m, None, 0.1, **ok)
    with pytest.raises(TypeError):
        gs().muon(p, g, m.half(), None, 0.1, **ok)
    with pytest.raises(RuntimeError, match="contiguous"):
        gs().muon(p.mT, g.mT, m.mT, None, 0.1, **ok)
    for valid in (torch.ones(5, dtype=torch.bool, device="cuda"), torch.ones(6, device="cuda"), torch.ones(6, 1, dtype=torch.bool, device="cuda")):
        with pytest.raises(ValueError, match="valid"):
            gs().muon(p, g, m, valid, 0.1, **ok)
    with pytest.raises(ValueError, match="valid"):
        gs().muon(p[0].contiguous(), g[0].contiguous(), m[0].contiguous(), torch.ones(4, dtype=torch.bool, device="cuda"), 0.1, **ok)
    with pytest.raises(RuntimeError, match="singular value"):
        gs().orthogonalize(p, coefficients=(2.0, 0.0, 0.0))


def test_param_used_by_a_living_graph_is_noticed():
    """A step in place counts as a modification: a backward pass that still needs the old values raises."""
    w = torch.nn.Parameter(torch.randn(20, 20, device="cuda"))
    loss = (w * w).sum()
    gs().muon(w, torch.randn(20, 20, device="cuda"), torch.zeros(20, 20, device="cuda"), None, 0.1, 0.9)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_muon_list_of_shapes_matches_one_by_one():
    shapes = [(64, 35), (64, 64), (64, 64), (3, 64), (200, 130), (9, 15, 3), (200, 130), (0, 4), (2, 200, 130), (130, 200), (64, 3), (35, 64),
              (2, 3, 130, 200), (3, 15, 9)]
    ps, grads, ms = ([data(s, torch.float32, 30 + 3 * i + j).cuda() for i, s in enumerate(shapes)] for j in range(3))
    alone = [(p.clone(), m.clone()) for p, m in zip(ps, ms)]
    lrs = [0.01 * (i + 1) for i in range(len(shapes))]
    gs().muon(ps, grads, ms, None, lrs, 0.95, 0.01)
    for (p, m), g, lr, got, got_m in zip(alone, grads, lrs, ps, ms):
        gs().muon(p, g, m, None, lr, 0.95, 0.01)
        assert torch.equal(p, got) and torch.equal(m, got_m)


def test_muon_many_tensors():
    """More tensors of a shape than one launch takes, or one slice of the list."""
    for shape in ((3, 3), (20, 24)):
        ps, grads, ms = ([data(shape, torch.float32, 100 + 3 * i + j, 0.1) for i in range(300)] for j in range(3))
        tp, tm = [p.cuda() for p in ps], [m.cuda() for m in ms]
        gs().muon(tp, [g.cuda() for g in grads], tm, None, 0.02, 0.9)
        for i in (0, 31, 32, 63, 64, 70, 255, 256, 299):
            check_step(ps[i], grads[i], ms[i], tp[i].cpu(), tm[i].cpu(), None, 0.02, 0.9, 0.0, True)


def test_muon_optimizer():
    """Three steps of the class on a decoder, per-splat SH bands under a visibility mask, and a checkpoint."""
    opt_args = dict(lr=0.02, momentum=0.9, weight_decay=0.1, adjust_lr_fn="match_rms_adamw")
    ps = [torch.nn.Parameter(data(s, torch.float32, 40 + i, 0.05).cuda()) for i, s in enumerate([(20, 8), (32, 64), (20, 8)])]
    opt = gs().Muon(ps, **opt_args)
    ref = [p.detach().cpu().double() for p in ps]
    bufs = [torch.zeros_like(r) for r in ref]
    for it in range(3):
        for i, p in enumerate(ps):
            p.grad = data(tuple(p.shape), torch.float32, 50 + 10 * it + i).cuda()
        versions = [p._version for p in ps]
        opt.step()
        assert all(p._version > v for p, v in zip(ps, versions))
        for i, p in enumerate(ps):
            lr = 0.02 * 0.2 * max(p.shape) ** 0.5
            ref[i], bufs[i] = step64(ref[i], p.grad.cpu(), bufs[i], None, lr, 0.9, 0.1, True)
            # 32-bit accuracy: gradients of singular values within 1 / 50 of the largest, amplified 485 times at most
            assert N.distance(p.detach().cpu(), ref[i]) < (it + 1) * 485 * 2.0**-21 * lr
    sh = torch.nn.Parameter(data((30, 15, 3), torch.float32, 60).cuda())
    opt = gs().Muon([sh], lr=0.01)
    before = sh.detach().clone()
    sh.grad = data((30, 15, 3), torch.float32, 61).cuda()
    vis = torch.arange(30, device="cuda") % 2 == 0
    opt.step(vis)
    assert torch.equal(sh.detach()[~vis], before[~vis]) and (sh.detach()[vis] != before[vis]).flatten(1).any(1).all()
    assert (opt.state[sh]["momentum_buffer"][~vis] == 0).all()
    other = gs().Muon([torch.nn.Parameter(sh.detach().clone())], lr=0.5)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    q = other.param_groups[0]["params"][0]
    q.grad = sh.grad.clone()
    opt.step(vis)
    other.step(vis)
    assert torch.equal(q.detach(), sh.detach())


def test_captured_step_and_gradient_replay():
    """Captured in a graph, a step replays on new gradients as the eager call does, beside another captured call."""
    side = torch.cuda.Stream()
    for shape in ((40, 15, 3), (2, 60, 50), (1, 300, 200)):
        p, g, m = (data(shape, torch.float32, s, 0.02).cuda() for s in (70, 71, 72))
        x = data(shape, torch.float32, 73).cuda().requires_grad_(True)
        v = data(shape, torch.float32, 74, 1.0).cuda()
        p0, m0 = p.clone(), m.clone()
        with torch.cuda.stream(side):
            gs().muon(p, g, m, None, 0.1, 0.9)
            torch.autograd.grad(gs().orthogonalize(x), x, v)
        side.synchronize()
        first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(first, stream=side):
            gs().muon(p, g, m, None, 0.1, 0.9)
        with torch.cuda.graph(second, stream=side):
            y = gs().orthogonalize(x)
            (v_x,) = torch.autograd.grad(y, x, v)
        p.copy_(p0), m.copy_(m0)
        g.copy_(data(shape, torch.float32, 75, 0.02))
        with torch.no_grad():
            x.copy_(data(shape, torch.float32, 76))
        first.replay(), second.replay()
        torch.cuda.synchronize()
        gs().muon(p0, g, m0, None, 0.1, 0.9)
        assert torch.equal(p, p0) and torch.equal(m, m0)
        z = gs().orthogonalize(x)
        assert torch.equal(y, z) and torch.equal(v_x, torch.autograd.grad(z, x, v)[0])


def test_other_stream():
    x = data((1, 400, 300), torch.float32, 80).cuda()
    want = gs().orthogonalize(x)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(gs().orthogonalize(x))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_splats_trained_with_both_optimizers():
    """A render's gradients through both: Adam for the geometry, Muon for the SH bands of what the camera sees."""
    from tests import _data

    d = _data.to(_data.scene(500, seed=1, width=64, height=48, fx=60.0), torch.device("cuda"))
    means = torch.nn.Parameter(d["means"].clone())
    sh0, shn = (torch.nn.Parameter(t.contiguous()) for t in (d["sh"][:, :1].clone(), d["sh"][:, 1:].clone()))
    adam = gs().SelectiveAdam([{"params": [means], "lr": 1e-4}, {"params": [sh0], "lr": 1e-3}], eps=1e-15, betas=(0.9, 0.999))
    opt = gs().Muon([shn], lr=1e-3, weight_decay=0.0)
    colors, _, meta = gs().rasterization(means, d["quats"], d["scales"], d["opacities"], torch.cat([sh0, shn], 1),
                                         d["viewmats"], d["Ks"], 64, 48, sh_degree=3, packed=False)
    colors.square().mean().backward()
    vis = (meta["radii"] > 0).all(-1).any(0)
    before, g = shn.detach().cpu().clone(), shn.grad.cpu()
    adam.step(vis)
    opt.step(vis)
    vis = vis.cpu()
    lr = 1e-3 * math.sqrt(shn.shape[1] / 3)
    want, _ = step64(before, g, torch.zeros_like(before), vis, lr, 0.95, 0.0, True)
    assert torch.equal(shn.detach().cpu()[~vis], before[~vis])
    # matrices whose gradient is below eps or of rank one keep 32-bit accuracy too: 485 is the steps' largest slope
    assert (shn.detach().cpu().double() - want).abs().max() <= 485 * 2.0**-21 * lr + 2.0**-24 * float(before.abs().max())
