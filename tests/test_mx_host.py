"""Microscaled matrices without a GPU: sizes of the layout, and the tests' own 64-bit reference
against values worked out by hand."""
import numpy as np
import pytest

import mx_reference as mx
from voxelengine import cuda as cu


@pytest.mark.parametrize("rows,cols,codes4,codes8,scales", [
    (1, 1, 64, 128, 512), (1, 128, 64, 128, 512), (1, 129, 128, 256, 1024), (128, 576, 128 * 320, 128 * 640, 5 * 512),
    (129, 576, 129 * 320, 129 * 640, 10 * 512), (0, 576, 0, 0, 0),
    (200000, 65536, 200000 * 32768, 200000 * 65536, 1563 * 512 * 512),
])
def test_sizes(rows, cols, codes4, codes8, scales):
    assert cu.mx_code_bytes(cu.MX_FP4, rows, cols) == codes4
    assert cu.mx_code_bytes(cu.MX_FP8, rows, cols) == codes8
    assert cu.mx_scale_bytes(rows, cols) == scales
    assert cu.mx_code_bytes(5, rows, cols) == 0


def test_scale_tile_offsets_cover_each_byte_once():
    off = mx.scale_offsets(256, 300)
    assert sorted(off.ravel()) == list(range(cu.mx_scale_bytes(256, 300)))
    assert off[33, 5] == 512 + 16 + 4 + 1 and off[128, 0] == 3 * 512


def test_reference_grids():
    assert list(mx.GRID[mx.FP4]) == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    assert mx.GRID[mx.FP8][1] == 2.0 ** -9 and mx.GRID[mx.FP8][-1] == 448 and mx.GRID[mx.FP8][8] == 2.0 ** -6
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0])
    assert list(mx.GRID[mx.FP4][mx.round_to_grid(ties, mx.FP4)]) == [0, 1, 1, 2, 2, 4, 4, 6]


def test_reference_block():
    x = np.zeros((1, 40))
    x[0, :4] = [7.0, -3.0, 0.4, -0.1]
    code, byte = mx.quantize(x, mx.FP4)
    assert byte[0, 0] == 127 and byte[0, 1] == 0        # floor(log2 7) - 2 = 0; an empty block
    assert list(mx.values(code, byte, 40, mx.FP4)[0, :4]) == [6.0, -3.0, 0.5, 0.0]
    x[0, 5] = np.inf
    code, byte = mx.quantize(x, mx.FP4)
    assert byte[0, 0] == 255 and np.isnan(mx.values(code, byte, 40, mx.FP4)[0, :32]).all()
