"""CPU checks of orthogonalize(), muon() and Muon: what they refuse, before any kernel is launched."""

import ctypes
import math

import pytest
import torch

import gsplat_b200
from tests import _newton_schulz as N


def test_refusals_of_orthogonalize():
    x = torch.randn(4, 4)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        gsplat_b200.orthogonalize(x)
    with pytest.raises(ValueError, match="M, N"):
        gsplat_b200.orthogonalize(torch.randn(4))
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        gsplat_b200.orthogonalize(x.double())
    for steps in (0, 33):
        with pytest.raises(ValueError, match="steps"):
            gsplat_b200.orthogonalize(x, steps=steps)
    for coefficients in ((1.5, -0.5), [(1.5, -0.5, 0.0)] * 4, [(1.5, -0.5)] * 5):
        with pytest.raises(ValueError, match="coefficients"):
            gsplat_b200.orthogonalize(x, coefficients=coefficients)
    for eps in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError, match="eps"):
            gsplat_b200.orthogonalize(x, eps=eps)


def test_refusals_of_muon():
    p, g, m = torch.randn(4, 4), torch.randn(4, 4), torch.zeros(4, 4)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        gsplat_b200.muon(p, g, m, None, 0.1, 0.9)
    with pytest.raises(ValueError, match="same length"):
        gsplat_b200.muon([p], [g], [], None, 0.1, 0.9)
    with pytest.raises(ValueError, match="same length"):
        gsplat_b200.muon([p], [g], [m], None, [0.1, 0.2], 0.9)
    with pytest.raises(ValueError, match="momentum"):
        gsplat_b200.muon(p, g, m, None, 0.1, 1.0)
    gsplat_b200.muon([], [], [], None, 0.1, 0.9)  # nothing to do


def test_refusals_of_the_optimizer():
    p = torch.nn.Parameter(torch.randn(4, 4))
    for bad in (dict(lr=-1.0), dict(weight_decay=-0.1), dict(adjust_lr_fn="other")):
        with pytest.raises(ValueError):
            gsplat_b200.Muon([p], **bad)
    with pytest.raises(ValueError, match="matrices"):
        gsplat_b200.Muon([torch.nn.Parameter(torch.randn(4))])
    gsplat_b200.Muon([p]).step()  # no gradient: nothing to do


def lib():
    from gsplat_b200.cuda import _backend

    return _backend.lib()


def triples(*c):
    flat = [v for t in c for v in t]
    return (ctypes.c_float * len(flat))(*flat)


def test_c_entry_points_refuse_before_any_launch():
    L, c = lib(), triples(*[N.QUINTIC] * 5)

    def fwd(batch=1, rows=8, cols=8, dtype=0, steps=5, co=c, eps=1e-7, kept=None, kept_size=0, scratch=None, size=0):
        return L.gsb_orthogonalize_fwd(batch, rows, cols, dtype, None, None, steps, co, eps, kept, kept_size, scratch, size, None)

    assert fwd(batch=-1) == -1 and b"negative" in L.gsb_last_error()
    assert fwd(dtype=3) == -2 and b"dtype" in L.gsb_last_error()
    assert fwd(steps=0) == -1 and fwd(steps=33) == -1 and b"steps" in L.gsb_last_error()
    assert fwd(co=None) == -1 and b"no coefficients" in L.gsb_last_error()
    assert fwd(eps=0.0) == -1 and fwd(eps=math.nan) == -1 and b"eps" in L.gsb_last_error()
    assert fwd(co=triples(*[(math.inf, 0.0, 0.0)] * 5)) == -1 and b"finite" in L.gsb_last_error()
    # 2^5 at a singular value of 1
    assert fwd(co=triples(*[(2.0, 0.0, 0.0)] * 5)) == -1 and b"32" in L.gsb_last_error()
    # the peak lies inside: 12 s - 12 s^3 is 0 at 1 and 4.6 at 0.58, and grows from there
    assert fwd(co=triples(*[(12.0, -12.0, 0.0)] * 5)) == -1
    assert fwd(rows=200, cols=200) == -1 and b"scratch" in L.gsb_last_error()
    assert fwd(rows=200, cols=200, kept=4096, kept_size=100) == -1 and b"kept" in L.gsb_last_error()
    assert fwd(batch=0) == 0 and fwd(rows=0) == 0 and fwd(cols=0) == 0
    rc = L.gsb_orthogonalize_bwd(1, 200, 200, 0, None, None, None, 5, c, 1e-7, None, 0, None, 0, None)
    assert rc == -1 and b"scratch" in L.gsb_last_error()
    def muon(n=0, tensors=None, dtype=0, state=0, scratch=None, size=0):
        return L.gsb_muon(n, tensors, dtype, state, None, 0.9, 1, 5, c, 1e-7, scratch, size, None)

    assert muon(n=1) == -1 and b"no tensor list" in L.gsb_last_error()
    assert muon(n=-1) == -1 and b"negative" in L.gsb_last_error()
    assert muon(state=1) == -2 and b"momentum buffer" in L.gsb_last_error()
    assert muon(dtype=1) == 0  # nothing to do
    from gsplat_b200.cuda._backend import GsbMuonTensor

    big = (GsbMuonTensor * 2)((None, None, None, 1, 200, 300, 1, 0.1, 1.0), (None, None, None, 0, 300, 200, 1, 0.1, 1.0))
    assert muon(2, big) == -1 and b"scratch" in L.gsb_last_error()
    assert L.gsb_muon_scratch_bytes(2, big, 0, 5) == L.gsb_orthogonalize_scratch_bytes(1, 200, 300, 0, 5, 0, 0)
    for bad in ((None, None, None, -1, 8, 8, 1, 0.1, 1.0), (None, None, None, 1, -8, 8, 1, 0.1, 1.0), (None, None, None, 1, 8, 8, 0, 0.1, 1.0)):
        assert muon(1, (GsbMuonTensor * 1)(bad)) == -1 and b"tensor 0" in L.gsb_last_error()


def test_scratch_sizes():
    L = lib()
    def size(batch, rows, cols, dtype, steps, backward, kept=0):
        return L.gsb_orthogonalize_scratch_bytes(batch, rows, cols, dtype, steps, backward, kept)

    kept = L.gsb_orthogonalize_kept_bytes
    assert size(1000000, 15, 3, 0, 5, 0) == 0 and size(10, 3, 128, 1, 5, 1) == 0  # thin
    assert size(10, 64, 64, 0, 5, 0) == 0 and size(10, 64, 64, 0, 5, 1) > 0  # on chip, forward
    assert size(10, 129, 129, 0, 5, 0) > 0 and size(0, 200, 200, 0, 5, 0) == 0
    assert size(1, 512, 256, 0, 5, 0) == size(1, 256, 512, 0, 5, 0)
    assert size(1, 256, 256, 0, 5, 1) > size(1, 256, 256, 0, 5, 1, 1)
    assert kept(10, 3, 15, 5) == 0 and kept(1, 256, 256, 5) > 0 and kept(1, 64, 64, 5) > 0
    # a large batch is taken in pieces: the scratch stays near 1 GiB, and nothing is kept
    assert size(100000, 512, 512, 0, 5, 0) < 1.1 * 2**30 and kept(100000, 512, 512, 5) == 0


def test_model_of_roundings_is_small_and_grows_with_them():
    """The tests' tolerances: without rounding the model is exact, 22 bits stay below 1e-3 for a matrix without tiny
    singular values, and 11 bits are further off than 22."""
    x = torch.randn(1, 150, 200)
    assert N.distance(N.newton_schulz(x), N.newton_schulz(x, products=0.0)) == 0
    fine = N.tolerance(x, 5, N.QUINTIC)
    assert 2.0**-24 < fine < 1e-3
    assert N.tolerance(x.bfloat16(), 5, N.QUINTIC) > fine
