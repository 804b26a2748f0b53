"""Microscaled SwiGLU products over matrices whose up half starts inside a scale tile."""
import numpy as np
import pytest

import mx_reference as mx
from test_gpu_mx import Mx, ctx, release  # noqa: F401 (fixtures)
from voxelengine import cuda as cu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def large(ctx):  # noqa: F811
    """[gate; up] of 2 x 65600 rows x 4096 columns: scales of more than 16 MiB with the halves apart."""
    rng = np.random.default_rng(0)
    ff, cols = 65600, 4096
    codes = rng.integers(0, 256, (2 * ff, cols // 2), dtype=np.uint8)
    byte = rng.integers(118, 122, (2 * ff, cols // 32), dtype=np.uint8)
    tiles = np.full((-(-2 * ff // 128), cols // 128, 32, 4, 4), 0xA5, np.uint8)  # tile row, tile, row % 32, row / 32, block
    rows = np.zeros((len(tiles) * 128, cols // 32), np.uint8)
    rows[:2 * ff] = byte
    tiles[:] = rows.reshape(len(tiles), 4, 32, cols // 128, 4).transpose(0, 3, 2, 1, 4)
    first = len(ctx._bufs)
    m = cu.MxMatrix(ctx.buffer(codes.size).upload(codes).ptr, ctx.buffer(tiles.size).upload(tiles).ptr, 2 * ff, cols, mx.FP4)
    held = ctx._bufs[first:]
    del ctx._bufs[first:]  # kept for the module
    yield m, codes, byte
    for b in held:
        b.free()


@pytest.mark.parametrize("n", [1, 2])
def test_swiglu_of_few_tokens_over_a_large_matrix(ctx, large, n):
    W, codes, byte = large
    ff, cols = W.rows // 2, W.cols
    rng = np.random.default_rng(n)
    xc, xb = mx.quantize(rng.standard_normal((n, cols)) * 0.1, mx.FP8)
    X, out = Mx(ctx, n, cols, mx.FP8, xc, xb), Mx(ctx, n, ff, mx.FP8)
    ctx.mx_gemm(cu.MxGemmArgs(w=W, x=X.m, epilogue=cu.EPI_SWIGLU, out=out.m))
    code, scale = out.get()
    x = mx.values(xc, xb, cols, mx.FP8)
    got = mx.values(code, scale, ff, mx.FP8)
    for c in (0, 32736, ff - 64):  # whole blocks, first and last ones among them
        g, u = (x @ mx.values(codes[r], byte[r], cols, mx.FP4).T for r in (slice(c, c + 64), slice(ff + c, ff + c + 64)))
        y = g / (1 + np.exp(-g)) * u
        s = np.repeat(np.exp2(scale[:, c // 32:c // 32 + 2].astype(np.float64) - 127), 32, 1)
        # Half a step of E4M3, its limit of 448, and fp32 sums (under 2^-16 of any of these values' scale).
        bound = np.maximum(np.abs(y) * 2.0 ** -4, 2.0 ** -10 * s) * (1 + 2.0 ** -10) + np.where(np.abs(y) > 447 * s, 64 * s, 0)
        assert (np.abs(got[:, c:c + 64] - y) <= bound + 2.0 ** -16 * 448 * s).all()


def test_swiglu_of_more_tokens_names_its_limit(ctx, large):
    """Refused before any launch: the workspace holds 16 MiB of sorted scales."""
    W = large[0]
    X, out = Mx(ctx, 3, W.cols, mx.FP8), Mx(ctx, 3, W.rows // 2, mx.FP8)
    with pytest.raises(cu.OpureError) as e:
        ctx.mx_gemm(cu.MxGemmArgs(w=W, x=X.m, epilogue=cu.EPI_SWIGLU, out=out.m))
    assert e.value.status == cu.ERR_UNSUPPORTED
