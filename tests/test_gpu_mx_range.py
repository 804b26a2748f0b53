"""Microscaled products at the ends of their types' ranges."""
import numpy as np
import pytest

import mx_reference as mx
from test_gpu_mx import FORMATS, Mx, Rows, ctx, product_bound, release  # noqa: F401 (fixtures)
from voxelengine import cuda as cu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 2, 3, 24, 300])
@pytest.mark.parametrize("fmt", FORMATS)
def test_scales_that_cancel(ctx, fmt, n):
    """A token's and a weight row's scales of one block as far apart as bytes go, their product
    near 1: no order of the multiplications may leave fp32's range."""
    rng = np.random.default_rng(n)
    rows, blocks = 72, 24
    cols = 32 * blocks
    centre = np.resize([1, 254, 20, 240, 127, 250, 90, 5], blocks)
    xb = np.broadcast_to(centre, (n, blocks))
    wb = np.clip(254 - centre + rng.integers(-3, 4, (rows, blocks)), 0, 254)
    codes = rng.integers(0, 256, (n, cols))
    xc = codes % 16 if fmt == mx.FP4 else np.where(codes % 128 == 127, 0, codes)
    wc = rng.integers(0, 16, (rows, cols))
    xc, wc = (xc[:, ::2] | xc[:, 1::2] << 4 if fmt == mx.FP4 else xc).astype(np.uint8), (wc[:, ::2] | wc[:, 1::2] << 4).astype(np.uint8)
    X, W = Mx(ctx, n, cols, fmt, xc, xb.astype(np.uint8)), Mx(ctx, rows, cols, mx.FP4, wc, wb.astype(np.uint8))
    Y = Rows(ctx, n, rows, "f32")
    ctx.mx_gemm(cu.MxGemmArgs(w=W.m, x=X.m, y=Y.ptr, y_type=cu.F32, y_stride=rows))
    x, w = mx.values(xc, xb, cols, fmt), mx.values(wc, wb, cols, mx.FP4)
    y = x @ w.T
    assert (np.abs(Y.get() - y) <= product_bound(x, w, y, "f32")).all()


@pytest.mark.parametrize("n", [1, 2, 24, 300])
@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_of_every_magnitude(ctx, fmt, n):
    """Each token and each weight row with a power of two of its own, results from 2^-100 to 2^100."""
    rng = np.random.default_rng(n)
    rows, cols = 96, 256
    x = rng.standard_normal((n, cols)) * np.exp2(np.linspace(-50, 50, n))[:, None]
    w = rng.standard_normal((rows, cols)) * np.exp2(np.linspace(-50, 50, rows))[:, None]
    (xc, xb), (wc, wb) = mx.quantize(x, fmt), mx.quantize(w, mx.FP4)
    X, W = Mx(ctx, n, cols, fmt, xc, xb), Mx(ctx, rows, cols, mx.FP4, wc, wb)
    Y = Rows(ctx, n, rows, "f32")
    ctx.mx_gemm(cu.MxGemmArgs(w=W.m, x=X.m, y=Y.ptr, y_type=cu.F32, y_stride=rows))
    xv, wv = mx.values(xc, xb, cols, fmt), mx.values(wc, wb, cols, mx.FP4)
    y = xv @ wv.T
    assert (np.abs(Y.get() - y) <= product_bound(xv, wv, y, "f32")).all()
