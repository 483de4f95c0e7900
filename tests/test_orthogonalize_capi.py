"""CPU checks of what the C entry points refuse before any launch: a kept state where there is none or that is too short, and lists
that do not agree."""

import ctypes

import pytest
import torch

from tests import _newton_schulz as N

# the calls carry pointers to nothing: only where no GPU could follow them
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="for machines without a GPU")


def lib():
    from gsplat_b200.cuda import _backend

    return _backend.lib()


# with a valid scratch size and pointers that are never followed: only the refusal keeps these calls from a launch
SOMEWHERE = 1 << 20


def both(batch, rows, cols, kept, size):
    L, c = lib(), (ctypes.c_float * 15)(*(list(N.QUINTIC) * 5))
    fwd = L.gsb_orthogonalize_fwd(batch, rows, cols, 0, None, None, 5, c, 1e-7, kept, size, SOMEWHERE, 1 << 40, None)
    message = L.gsb_last_error()
    bwd = L.gsb_orthogonalize_bwd(batch, rows, cols, 0, None, None, None, 5, c, 1e-7, kept, size, SOMEWHERE, 1 << 40, None)
    return fwd, bwd, message


@pytest.mark.parametrize("batch,rows,cols", [(1, 4096, 4096), (100000, 512, 512), (10, 15, 3)])
@pytest.mark.parametrize("size", [1, 16, 1 << 33])
def test_kept_state_where_there_is_none(batch, rows, cols, size):
    """Above 1 GiB with the scratch, and for thin matrices, none is kept, whatever room the caller offers."""
    assert lib().gsb_orthogonalize_kept_bytes(batch, rows, cols, 5) == 0
    fwd, bwd, message = both(batch, rows, cols, SOMEWHERE, size)
    assert fwd == -1 and bwd == -1 and b"no state is kept" in message


@pytest.mark.parametrize("batch,rows,cols", [(1, 300, 300), (8, 64, 64)])
def test_kept_state_too_short(batch, rows, cols):
    needed = lib().gsb_orthogonalize_kept_bytes(batch, rows, cols, 5)
    for size in (0, 1, needed - 1):
        fwd, bwd, message = both(batch, rows, cols, SOMEWHERE, size)
        assert fwd == -1 and bwd == -1 and b"needs %d" % needed in message


def test_gains_of_a_muon_list_must_agree():
    from gsplat_b200.cuda._backend import GsbMuonTensor

    L, c = lib(), (ctypes.c_float * 15)(*(list(N.QUINTIC) * 5))
    for other in (0.0, 0.2, float("nan")):
        two = (GsbMuonTensor * 2)((None, None, None, 0, 4, 4, 1, 0.1, 1.0, 0.1), (None, None, None, 0, 4, 4, 1, 0.1, 1.0, other))
        assert L.gsb_muon(2, two, 0, 0, None, 0.9, 1, 5, c, 1e-7, None, 0, None) == -1 and b"gain" in L.gsb_last_error()


def test_scratch_of_a_forward_that_keeps_its_state():
    """X, A and B lie in the state: beside it only the norm's sums are needed."""
    size = lib().gsb_orthogonalize_scratch_bytes
    assert size(1, 3000, 2900, 0, 5, 0, 0) > 100 * 2**20
    assert size(1, 3000, 2900, 0, 5, 0, 1) < 2**16
    assert size(1, 300, 200, 0, 5, 1, 1) > 2**20 // 4  # backwards G, S and T are


@pytest.mark.parametrize("rows,cols", [(1, 1_100_000_000), (1_999_999_999, 1), (5000, 128), (128, 4097)])
def test_sizes_of_long_matrices(rows, cols):
    """Far beyond what a cluster holds, where its size was searched for without end; the scratch holds two X as pairs of halves."""
    x = -(-max(rows, cols) // 8) * 8 * min(rows, cols)
    assert 8 * x < lib().gsb_orthogonalize_scratch_bytes(1, rows, cols, 1, 5, 0, 0) < 8 * x + 2**20
    assert lib().gsb_orthogonalize_tile(1, rows, cols, 1, 0, 0, 148) > 0


def test_sides_that_do_not_fit_are_refused():
    from gsplat_b200.cuda._backend import GsbMuonTensor

    L, c, side = lib(), (ctypes.c_float * 15)(*(list(N.QUINTIC) * 5)), 2_000_000_001
    for rows, cols in ((1, side), (side, 1), (1, 2**31 - 1)):
        assert L.gsb_orthogonalize_scratch_bytes(1, rows, cols, 0, 5, 0, 0) == 0 and L.gsb_orthogonalize_kept_bytes(1, rows, cols, 5) == 0
        for f, pointers in ((L.gsb_orthogonalize_fwd, 2), (L.gsb_orthogonalize_bwd, 3)):
            rc = f(1, rows, cols, 0, *[None] * pointers, 5, c, 1e-7, None, 0, SOMEWHERE, 1 << 40, None)
            assert rc == -1 and b"a side may" in L.gsb_last_error()
        one = (GsbMuonTensor * 1)((None, None, None, 1, rows, cols, 1, 0.1, 1.0))
        assert L.gsb_muon(1, one, 0, 0, None, 0.9, 1, 5, c, 1e-7, SOMEWHERE, 1 << 40, None) == -1
    import gsplat_b200

    # a size of 2^32 + 3 would otherwise pass for 3
    for shape in ((1, 2**32 + 3), (2**32 + 3, 1), (2, 1, side)):
        with pytest.raises(ValueError, match="a side may"):
            gsplat_b200.orthogonalize(torch.zeros(1).expand(shape))


def test_missing_and_misplaced_pointers_are_refused():
    from gsplat_b200.cuda._backend import GsbMuonTensor

    L, c = lib(), (ctypes.c_float * 15)(*(list(N.QUINTIC) * 5))

    def fwd(rows, cols, dtype, x, y, scratch=SOMEWHERE, kept=None):
        size = L.gsb_orthogonalize_kept_bytes(1, rows, cols, 5) if kept else 0
        return L.gsb_orthogonalize_fwd(1, rows, cols, dtype, x, y, 5, c, 1e-7, kept, size, scratch, 1 << 40, None)

    def bwd(rows, cols, dtype, x, v, out, scratch=SOMEWHERE):
        return L.gsb_orthogonalize_bwd(1, rows, cols, dtype, x, v, out, 5, c, 1e-7, None, 0, scratch, 1 << 40, None)

    for rows, cols in ((15, 3), (3, 60), (40, 50), (300, 200)):
        for bad in (None, SOMEWHERE + 1, SOMEWHERE + 2):
            want = b"missing" if bad is None else b"between"
            assert fwd(rows, cols, 0, bad, SOMEWHERE) == -1 and want in L.gsb_last_error()
            assert fwd(rows, cols, 0, SOMEWHERE, bad) == -1 and want in L.gsb_last_error()
            for i in range(3):
                p = [SOMEWHERE] * 3
                p[i] = bad
                assert bwd(rows, cols, 0, *p) == -1 and want in L.gsb_last_error()
        assert fwd(rows, cols, 1, SOMEWHERE + 1, SOMEWHERE) == -1 and b"between" in L.gsb_last_error()
    assert fwd(300, 200, 0, SOMEWHERE, SOMEWHERE, scratch=SOMEWHERE + 8) == -1 and b"16 bytes" in L.gsb_last_error()
    assert fwd(300, 200, 0, SOMEWHERE, SOMEWHERE, kept=SOMEWHERE + 8) == -1 and b"16 bytes" in L.gsb_last_error()
    assert bwd(40, 50, 0, SOMEWHERE, SOMEWHERE, SOMEWHERE, scratch=SOMEWHERE + 4) == -1 and b"16 bytes" in L.gsb_last_error()
    for i in range(3):
        for bad, state in ((None, 0), (SOMEWHERE + 2, 0), (SOMEWHERE + 1, 1)):
            p = [SOMEWHERE] * 3
            p[i] = bad
            one = (GsbMuonTensor * 1)((*p, 1, 4, 4, 1, 0.1, 1.0))
            assert L.gsb_muon(1, one, state, state, None, 0.9, 1, 5, c, 1e-7, None, 0, None) == -1
            assert (b"missing" if bad is None else b"between") in L.gsb_last_error()
