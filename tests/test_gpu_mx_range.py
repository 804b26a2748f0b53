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


@pytest.mark.parametrize("n", [1, 24, 300])
@pytest.mark.parametrize("out_fmt", FORMATS)
def test_swiglu_of_far_negative_gates(ctx, out_fmt, n):
    """silu(g) is g exp(g) there, a normal fp32 number down to g = -92; an up value of 2^100 makes
    the product an ordinary one. Gates are sums of three codes with scales of their own, exact."""
    rng = np.random.default_rng(5)
    gates, cols = [-72.0, -84.0, -88.0, -90.0, -1.5], 128
    ff = 32 * len(gates)
    steps = np.sort(np.concatenate([[0], np.ravel(np.outer([1, 1.5], 2.0 ** np.arange(-3, 7)))]))
    w = np.zeros((2 * ff, cols))
    for j in range(ff):
        left = -gates[j // 32]
        for k in (0, 32, 64):
            part = steps[steps <= left][-1]
            w[j, k], left = -part, left - part
        assert left == 0
    w[ff:, 96] = 2.0 ** 100 * (1 + 0.5 * rng.integers(0, 2, ff))
    x = np.zeros((n, cols))
    x[:, ::32] = 1.0
    (wc, wb), (xc, xb) = mx.quantize(w, mx.FP4), mx.quantize(x, mx.FP8)
    assert np.array_equal(mx.values(wc, wb, cols, mx.FP4), w) and np.array_equal(mx.values(xc, xb, cols, mx.FP8), x)
    W, X, out = Mx(ctx, 2 * ff, cols, cu.MX_FP4, wc, wb), Mx(ctx, n, cols, cu.MX_FP8, xc, xb), Mx(ctx, n, ff, out_fmt)
    ctx.mx_gemm(cu.MxGemmArgs(w=W.m, x=X.m, epilogue=cu.EPI_SWIGLU, out=out.m))
    g, u = x @ w[:ff].T, x @ w[ff:].T
    y = g * np.exp(g) / (1 + np.exp(g)) * u
    want_code, want_byte = mx.quantize(y, out_fmt)
    # fp32's roundings, and exp(-90) as a subnormal, are off by 2^-19 at most; no value lies within
    # 2^-16 of a rounding boundary of its code or scale, so the bytes are the definition's.
    for f in (1 - 2.0 ** -16, 1 + 2.0 ** -16):
        assert all(np.array_equal(a, b) for a, b in zip(mx.quantize(y * f, out_fmt), (want_code, want_byte)))
    code, byte = out.get()
    assert np.array_equal(byte, want_byte)
    assert np.array_equal(code, want_code)
