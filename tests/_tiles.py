"""Shapes that between them take every kind of tile, for the tests of the tiled products, and what each takes on a B200."""

SMS = 148  # of a B200

# shape: tiles of A, B and X (of S, T and G too, in 32 bits) for float32, then of A, B and X for bfloat16: 1000 x the blocks that share
# the depth + the tile's columns. Sides that divide by no tile's, and more tiles than SMs for the persistent loops.
TILES = {
    (1, 700, 1300): ([4128, 1064, 1064], [1064, 1064, 1064]),
    (1, 1000, 4100): ([2064, 1064, 1256], [2064, 1064, 1256]),
    (1, 1100, 2300): ([2128, 1064, 1256], [2128, 1064, 1256]),
    (40, 300, 520): ([1128, 1128, 1128], [1128, 1128, 1128]),
    (300, 130, 150): ([1128, 1128, 1256], [1128, 1128, 1256]),
    (2, 1500, 1700): ([1256, 1256, 1256], [1256, 1256, 1256]),
    (1, 2050, 4100): ([1256, 1256, 1128], [1256, 1256, 1128]),
    (1, 2100, 17000): ([1256, 1256, 1256], [1128, 1256, 1256]),
}
