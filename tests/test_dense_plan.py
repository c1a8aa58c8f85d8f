"""Which kernel the 8-bit product takes for the shapes that the GPU tests run: every kernel is among them, with every number of rows of the
streamed one and every tile, whatever becomes of the table of costs."""
import ctypes

import pytest

FEW, STREAMED, TILES, ANY = "few rows", "streamed", "tiles", "tiles of any rows"

# rows x cols x inner, rows at multiples of 16 bytes: kernel, rows that it takes at once, whether the inner dimension is cut.
# Streamed: every number of rows, ragged ones; one tile of 16 columns for a workgroup, and two and three; stages in the steady
# part of its loop and too few for it; inner dimensions that end inside a stage, in its first and last piece.
SHAPES = {
    (3, 4100, 2048): (STREAMED, 16, False), (16, 8200, 4096): (STREAMED, 16, False), (9, 100, 16433): (STREAMED, 16, False),
    (16, 33, 4160): (STREAMED, 16, False), (5, 9001, 2111): (STREAMED, 16, False),
    (17, 4113, 2128): (STREAMED, 32, False), (32, 9000, 8192): (STREAMED, 32, False), (20, 40, 5000): (STREAMED, 32, False),
    (40, 130, 16400): (STREAMED, 48, False), (48, 9000, 4160): (STREAMED, 48, False), (33, 4097, 2049): (STREAMED, 48, False),
    (63, 4099, 2063): (STREAMED, 64, False), (64, 8200, 12288): (STREAMED, 64, False), (50, 20, 2110): (STREAMED, 64, False),
    (2, 500, 5000): (FEW, 16, False), (30, 700, 1900): (FEW, 32, False), (40, 300, 40000): (FEW, 48, True), (64, 1000, 2040): (FEW, 64, False),
    (4, 60, 100000): (FEW, 16, True),
    # tiles: whole ones and ragged edges, a last stage that is not whole, one after the cuts too
    (4000, 4090, 2100): (TILES, 256, False), (4096, 4096, 4096): (TILES, 256, False), (130, 8000, 60033): (TILES, 256, True),
    (4000, 3100, 257): (TILES, 128, False), (1500, 3100, 4000): (TILES, 128, False), (600, 500, 30001): (TILES, 128, True),
    (257, 300, 1111): (TILES, 64, False), (65, 600, 20001): (TILES, 64, True), (200, 200, 30011): (TILES, 64, True),
    (65, 129, 127): (ANY, 64, False), (2048, 6200, 160): (ANY, 128, False),
}
KERNELS = [FEW, STREAMED, TILES, ANY]   # enum geo_sc_q8_kernel


def plan(rows, cols, inner, x_stride, w_stride, x=4096, w=4096):
    from geo_amd import _native
    out = [ctypes.c_int() for _ in range(3)]
    assert _native.lib().geo_sc_matmul_q8_plan(x, x_stride, w, w_stride, rows, cols, inner, *[ctypes.byref(v) for v in out]) == 0
    return KERNELS[out[0].value], out[1].value, out[2].value > 1


@pytest.mark.parametrize("shape", SHAPES)
def test_kernel_of_the_shapes_that_are_tested(shape):
    stride = (shape[2] + 15) // 16 * 16
    assert plan(*shape, stride, stride) == SHAPES[shape]


def test_every_kernel_is_among_them():
    assert {v[:2] for v in SHAPES.values()} == {(STREAMED, r) for r in (16, 32, 48, 64)} | {(FEW, r) for r in (16, 32, 48, 64)} | \
        {(TILES, t) for t in (64, 128, 256)} | {(ANY, t) for t in (64, 128)}


def test_rows_at_other_addresses():
    # few rows are taken as they lie, tiles are laid out anew
    assert plan(48, 4096, 16384, 16385, 16384)[0] == FEW and plan(48, 4096, 16384, 16384, 16384, w=4097)[0] == FEW
    assert plan(4000, 4090, 2100, 2101, 2112) == plan(4000, 4090, 2100, 2112, 2112, x=4097) == (TILES, 256, False)


def test_refusals():
    from geo_amd import _native
    out = [ctypes.byref(ctypes.c_int()) for _ in range(3)]
    for sizes, strides in (((0, 1, 1), (16, 16)), ((1, 0, 1), (16, 16)), ((1, 1, 0), (16, 16)), ((1, 1, 131072), (16, 16)), ((1, 1, 1), (-1, 16)), ((1, 1, 1), (16, -1))):
        assert _native.lib().geo_sc_matmul_q8_plan(4096, strides[0], 4096, strides[1], *sizes, *out) == 1
    assert _native.lib().geo_sc_matmul_q8_plan(4096, 16, 4096, 16, 1, 1, 1, out[0], None, out[2]) == 1
