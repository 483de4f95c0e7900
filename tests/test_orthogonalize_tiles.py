"""CPU checks that the shapes of the GPU tests take the tiles that they are there for: a change of the tiles' measured costs must not
leave a kernel without a test."""

import pytest

from tests._tiles import SMS, TILES


def tiles(shape, dtype, products):
    from gsplat_b200.cuda import _backend

    return [_backend.lib().gsb_orthogonalize_tile(*shape, dtype, 0, q, SMS) for q in products]


@pytest.mark.parametrize("shape", TILES)
def test_tiles_of_a_shape(shape):
    split, hi = TILES[shape]
    assert tiles(shape, 0, range(3)) == split and tiles(shape, 2, range(3)) == split
    assert tiles(shape, 0, range(3, 6)) == split
    assert tiles(shape, 1, range(3)) == hi and tiles(shape, 1, range(3, 6)) == split
    turned = (shape[0], shape[2], shape[1])
    assert tiles(turned, 0, range(3)) == split


def test_every_tile_is_taken():
    """For each product 64, 128 and 256 columns, with hi + lo and hi alone, and a shared depth at 64 and 128 of the products
    that may share it (A, S)."""
    for dtype, products in ((0, range(6)), (1, range(3))):
        for q in products:
            taken = {tiles(shape, dtype, [q])[0] for shape in TILES}
            columns = {t % 1000 for t in taken}
            if q % 3 == 0:
                assert {t % 1000 for t in taken if t >= 2000} == {64, 128}
                columns |= {64}  # below that number of tiles the depth is shared
            assert columns == {64, 128, 256}, (dtype, q, taken)


def test_no_tiles_where_there_are_none():
    assert tiles((5, 15, 3), 0, range(6)) == [0] * 6  # thin
    assert tiles((5, 64, 64), 0, range(3)) == [0] * 3 and tiles((5, 64, 64), 0, [3]) == [1064]  # clustered, but not backwards
    assert tiles((5, 200, 200), 0, [-1, 6]) == [0, 0]


def test_deep_products_of_bfloat16_leave_the_pair():
    assert tiles((1, 16300, 16300), 1, range(3)) == [1256] * 3 and tiles((1, 16400, 16500), 1, range(3)) == [1128] * 3
    assert tiles((1, 16400, 16500), 0, range(3)) == [1256] * 3
