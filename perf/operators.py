"""Cases of the matrix-orthogonalising operators: ``orthogonalize``, its gradient, and the ``muon`` step.

``orthogonalize(x)`` divides each matrix by its Frobenius norm and takes ``steps`` Newton-Schulz steps
X <- a X + (b A + c A A) X with A = X X^T; ``muon`` keeps a momentum of the gradients, orthogonalises it
(Nesterov form) and takes the result, with a decoupled weight decay, from the parameters. Where ``own`` is
false the operators run in their plain form (elementary products in 32 bits, the norm summed in 64);
where it is true they are the calls of ``gsplat_b200``.
"""

import math

import torch

own = False

QUINTIC = (3.4445, -4.7750, 2.0315)  # the optimiser's steep polynomial
CUBIC = (1.5, -0.5, 0.0)  # converges to the orthogonal factor itself
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
MOMENTUM, WEIGHT_DECAY, LR, EPS = 0.95, 0.1, 1e-3, 1e-7
LARGEST = 4096  # the longest side of a drawn weight matrix


def listed():
    return [
        # the rotations of a training set's cameras, brought back to orthogonal ones: latency alone
        dict(name="rotations", op="orthogonalize", shapes="256x3x3", dtype="float32", steps=8, kind="rotation"),
        # the layers of a small feature decoder, stacked
        dict(name="decoder stack", op="orthogonalize", shapes="8x64x64", dtype="bfloat16", steps=5, kind="quintic"),
        # a matrix whose sides divide by nothing
        dict(name="odd matrix", op="orthogonalize", shapes="1x257x1000", dtype="float32", steps=5, kind="quintic"),
        # a wide projection of a transformer
        dict(name="wide projection", op="orthogonalize", shapes="1x2048x8192", dtype="bfloat16", steps=5, kind="quintic"),
        # a rotation for each splat, trained through its raw 3x3 matrix
        dict(name="splat rotations grad", op="gradient", shapes="100000x3x3", dtype="float32", steps=6, kind="rotation"),
        # mixing matrices held orthogonal while they are trained
        dict(name="mixing stack grad", op="gradient", shapes="4x256x1024", dtype="bfloat16", steps=5, kind="quintic"),
        dict(name="tall odd grad", op="gradient", shapes="1x1111x300", dtype="float32", steps=5, kind="quintic"),
        # the higher SH bands of a million splats, of which one camera sees a part
        dict(name="sh bands step", op="muon", shapes="1000000x15x3", dtype="float32", state="float32", visible=0.45),
        # a colour decoder's four layers: latency, and shapes of their own
        dict(name="decoder step", op="muon", shapes="1x64x35,1x64x64,1x64x64,1x3x64", dtype="float32", state="float32", visible=1.0),
        # one transformer block of 16-bit weights with its momentum in 32 bits
        dict(name="block step", op="muon", shapes="1x1024x1024,1x1024x1024,1x1024x1024,1x1024x1024,1x4096x1024,1x1024x4096",
             dtype="bfloat16", state="float32", visible=1.0),
        # per-head projections, tall and odd
        dict(name="heads step", op="muon", shapes="12x1000x77", dtype="float16", state="float16", visible=1.0),
        # a large square weight in 32 bits
        dict(name="large step", op="muon", shapes="1x4096x4096", dtype="float32", state="float32", visible=1.0),
    ]


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["orthogonalize", "gradient", "muon"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if rng.random() < 0.35:  # many thin matrices: a few numbers for each splat
        m, n = rng.randint(3, 25), rng.randint(2, 4)
        shapes = [(_log(rng, 1, 20000000 // (m * n)), m, n)]
    else:  # weights: one shape, or several of a model
        shapes = []
        for _ in range(1 if op != "muon" else rng.choice([1, 1, 2, 5])):
            while True:
                s = (rng.choice([1, 1, 2, 3, 7]), _log(rng, 5, LARGEST), _log(rng, 5, LARGEST))
                if _flops(s, 5) * 3 <= _flops((1, LARGEST, LARGEST), 5) / 2:
                    break
            shapes.append(s)
    case = dict(op=op, shapes=",".join("%dx%dx%d" % s for s in shapes), dtype=dtype)
    if op == "muon":
        thin = len(shapes) == 1 and shapes[0][0] > 1
        return dict(case, state=rng.choice([dtype, "float32"]), visible=rng.choice([1.0, 0.3, 0.7]) if thin else 1.0)
    return dict(case, steps=rng.randint(4, 6), kind="quintic")


def _matrices(gen, shape, kind):
    """Gradients as training meets them: a few directions that carry most of it, over noise; or near-rotations."""
    b, m, n = shape
    x = torch.randn(b, m, n, generator=gen, device="cuda")
    if kind == "rotation":
        q = torch.randn(b, 4, generator=gen, device="cuda")
        w, u, v, t = (q / q.norm(dim=-1, keepdim=True)).unbind(-1)
        r = torch.stack([1 - 2 * (v * v + t * t), 2 * (u * v - w * t), 2 * (u * t + w * v),
                         2 * (u * v + w * t), 1 - 2 * (u * u + t * t), 2 * (v * t - w * u),
                         2 * (u * t - w * v), 2 * (v * t + w * u), 1 - 2 * (u * u + v * v)], -1).reshape(b, 3, 3)
        return r + 0.05 * x
    r = max(1, min(m, n) // 16)
    signal = torch.randn(b, m, r, generator=gen, device="cuda") @ torch.randn(b, r, n, generator=gen, device="cuda")
    return 1e-4 * (x + signal / math.sqrt(r))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]
    shapes = _shapes(case)
    if case["op"] != "muon":
        x = _matrices(gen, shapes[0], case["kind"]).to(dtype)
        state = dict(op=case["op"], x=x, steps=case["steps"], coefficients=CUBIC if case["kind"] == "rotation" else QUINTIC)
        if case["op"] == "gradient":
            state["v"] = torch.randn(shapes[0], generator=gen, device="cuda").to(dtype)
        return state
    kept = DTYPES[case["state"]]
    params = [(torch.randn(s, generator=gen, device="cuda") * 0.02).to(dtype) for s in shapes]
    grads = [_matrices(gen, s, "gradient").to(dtype) for s in shapes]
    buffers = [(g.float() + _matrices(gen, s, "gradient")).mul_(0.5).to(kept) for g, s in zip(grads, shapes)]
    valid = None
    if case["visible"] < 1.0:
        valid = torch.rand(shapes[0][0], generator=gen, device="cuda") < case["visible"]
    # the step for each shape: the update's root mean square is that of an Adam step
    lrs = [LR * 0.2 * math.sqrt(max(s[1:])) for s in shapes]
    return dict(op="muon", params=params, grads=grads, buffers=buffers, valid=valid, lrs=lrs)


def _newton_schulz(x, steps, coefficients):
    """The plain form, in 32 bits, on the side that is shorter."""
    a, b, c = coefficients
    if x.shape[-2] > x.shape[-1]:
        return _newton_schulz(x.mT, steps, coefficients).mT
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt()
    x = (x.double() / norm.clamp_min(EPS)).float()
    for _ in range(steps):
        g = x @ x.mT
        x = a * x + (b * g + c * (g @ g)) @ x
    return x


def _plain_muon(param, grad, buffer, valid, lr):
    """One tensor's step in place; rows that `valid` leaves out keep their values."""
    at = slice(None) if valid is None else valid
    p, g, m = param[at].float(), grad[at].float(), buffer[at].float()
    m = m + (1 - MOMENTUM) * (g - m)
    update = _newton_schulz(g + MOMENTUM * (m - g), 5, QUINTIC)
    param[at] = (p * (1 - lr * WEIGHT_DECAY) - lr * update).to(param.dtype)
    buffer[at] = m.to(buffer.dtype)


def run(state):
    if own:
        import gsplat_b200

        if state["op"] == "muon":
            gsplat_b200.muon(state["params"], state["grads"], state["buffers"], state["valid"], state["lrs"], MOMENTUM, WEIGHT_DECAY)
            return {"params": state["params"], "buffers": state["buffers"]}
        x = state["x"].detach().requires_grad_(state["op"] == "gradient")
        y = gsplat_b200.orthogonalize(x, steps=state["steps"], coefficients=state["coefficients"])
        if state["op"] == "orthogonalize":
            return {"y": y}
        return {"y": y.detach(), "v_x": torch.autograd.grad(y, x, state["v"])[0]}
    if state["op"] == "muon":
        n = len(state["params"])
        list(map(_plain_muon, state["params"], state["grads"], state["buffers"], [state["valid"]] * n, state["lrs"]))
        return {"params": state["params"], "buffers": state["buffers"]}
    x = state["x"].detach().float().requires_grad_(state["op"] == "gradient")
    y = _newton_schulz(x, state["steps"], state["coefficients"])
    if state["op"] == "orthogonalize":
        return {"y": y.to(state["x"].dtype)}
    v_x = torch.autograd.grad(y, x, state["v"].float())[0]
    return {"y": y.detach().to(state["x"].dtype), "v_x": v_x.to(state["x"].dtype)}


def _exact(x, steps, coefficients):
    """64 bits, with the products on the other side: X <- X (a I + b G + c G^2), G = X^T X."""
    a, b, c = coefficients
    if x.shape[-2] < x.shape[-1]:
        return _exact(x.mT, steps, coefficients).mT
    x = x / torch.linalg.matrix_norm(x)[:, None, None].clamp_min(EPS)
    eye = torch.eye(x.shape[-1], dtype=torch.float64, device=x.device)
    for _ in range(steps):
        g = x.mT @ x
        x = x @ (a * eye + g @ (b * eye + c * g))
    return x


def exact(case, seed):
    state = prepare(case, seed)
    if state["op"] != "muon":
        x = state["x"].double().requires_grad_(state["op"] == "gradient")
        y = _exact(x, state["steps"], state["coefficients"])
        if state["op"] == "orthogonalize":
            return {"y": y}
        return {"y": y.detach(), "v_x": torch.autograd.grad(y, x, state["v"].double())[0]}
    params, buffers = [], []
    for p, g, m, lr in zip(state["params"], state["grads"], state["buffers"], state["lrs"]):
        p, g, m = p.double(), g.double(), m.double()
        new_m = MOMENTUM * m + (1 - MOMENTUM) * g
        update = _exact((1 - MOMENTUM) * g + MOMENTUM * new_m, 5, QUINTIC)
        new_p = p - lr * (WEIGHT_DECAY * p + update)
        if state["valid"] is not None:
            keep = state["valid"][:, None, None]
            new_m, new_p = torch.where(keep, new_m, m), torch.where(keep, new_p, p)
        params.append(new_p)
        buffers.append(new_m)
    return {"params": params, "buffers": buffers}


def _flops(shape, steps):
    """Of the iteration: A and A A are symmetric, and half of each is enough; (b A + c A A) X is whole."""
    b, m, n = shape[0], min(shape[1:]), max(shape[1:])
    return b * steps * (3 * m * m * n + m * m * m)


def work(case):
    size = {"float32": 4, "bfloat16": 2, "float16": 2}
    shapes = _shapes(case)
    numel = sum(b * m * n for b, m, n in shapes)
    if case["op"] == "muon":
        seen = case["visible"]
        # the parameter and its momentum are read and written, the gradient read
        moved = numel * seen * (3 * size[case["dtype"]] + 2 * size[case["state"]])
        return {"bytes": moved + (shapes[0][0] if seen < 1 else 0), "flops": seen * sum(_flops(s, 5) for s in shapes)}
    flops = _flops(shapes[0], case["steps"])
    if case["op"] == "orthogonalize":
        return {"bytes": 2 * numel * size[case["dtype"]], "flops": flops}
    # x, v and the two outputs; the backward's three symmetric halves and two whole products are twice the forward's
    return {"bytes": 4 * numel * size[case["dtype"]], "flops": 3 * flops}
