"""Which codes of the microscaled norm and SwiGLU may differ from the definition's: a result computed
with relative error r has another code than the exact one only if a rounding boundary lies within r
of it.
"""
import numpy as np
import pytest

import mx_reference as mx
from test_gpu_mx import Mx, Rows, ctx, release  # noqa: F401 (fixtures)
from voxelengine import cuda as cu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_norm(ctx, t):
    """One rounding of s = x + r in fp32 and one of the result (2^-24 each); the inverse root and its
    product with the gain are held as pairs, the squares added in fp32 only eight at a time: r = 2^-23.
    Boundaries of E4M3 codes are 2^-4 to 2^-3 of a value apart, so that 2 r / 2^-4 of these values at
    most are that near to one: 16. The limit is twice that and 4."""
    rng = np.random.default_rng(1)
    rows, cols = 2048, 2048
    X, R, out = Rows(ctx, rows, cols, t), Rows(ctx, rows, cols, t), Mx(ctx, rows, cols, mx.FP8)
    x, r = X.put(rng.standard_normal((rows, cols))), R.put(3 * rng.standard_normal((rows, cols)))
    gain = (1 + 0.1 * rng.standard_normal(cols)).astype(np.float16)
    ctx.mx_rmsnorm(cu.MxNormArgs(x=X.ptr, x_type=cu.VALUE_TYPES[t], x_stride=cols, residual=R.ptr, gain=ctx.to_device(gain).ptr, eps=1e-5,
                                 out=out.m))
    s = x + r
    want, scale = mx.quantize(s / np.sqrt((s * s).mean(1, keepdims=True) + 1e-5) * gain.astype(np.float64), mx.FP8)
    code, byte = out.get()
    assert np.count_nonzero(byte != scale) <= 1
    assert np.count_nonzero(code != want) <= 36


@pytest.mark.parametrize("n", [2, 64, 600])
def test_swiglu(ctx, n):
    """Products whose sums fp32 holds exactly (whole numbers of 1/8), so that the codes show silu and the
    multiplication alone: exp, 1 + t, a quotient and two products, each rounded to fp32, exp off by two
    more units: 2^-22 together. Gates from -70 to 70, so that exp's argument counts too. Many results
    (large gates, whose silu is all but the gate) lie next to a boundary, so each is asked for by itself."""
    rng = np.random.default_rng(n)
    ff, cols = 2048, 256
    w = rng.choice([-2, -1.5, -1, -0.5, 0, 0.5, 1, 1.5, 2], (2 * ff, cols))
    w[:, ::32] = rng.choice([-4, 4], (2 * ff, cols // 32))  # blocks' scales of 1
    x = rng.choice([-1, -0.5, -0.25, 0.25, 0.5, 1], (n, cols))
    (wc, wb), (xc, xb) = mx.quantize(w, mx.FP4), mx.quantize(x, mx.FP8)
    assert np.array_equal(mx.values(wc, wb, cols, mx.FP4), w) and np.array_equal(mx.values(xc, xb, cols, mx.FP8), x)
    W, X, out = Mx(ctx, 2 * ff, cols, mx.FP4, wc, wb), Mx(ctx, n, cols, mx.FP8, xc, xb), Mx(ctx, n, ff, mx.FP8)
    ctx.mx_gemm(cu.MxGemmArgs(w=W.m, x=X.m, epilogue=cu.EPI_SWIGLU, out=out.m))
    g, u = x @ w[:ff].T, x @ w[ff:].T
    y, r = g / (1 + np.exp(-g)) * u, 2.0 ** -22
    code, byte = out.get()
    (low, low_byte), (high, high_byte) = mx.quantize(y * (1 - r), mx.FP8), mx.quantize(y * (1 + r), mx.FP8)
    assert ((byte == low_byte) | (byte == high_byte)).all()
    same = np.repeat(low_byte == high_byte, 32, 1)  # the scale is settled
    assert same.mean() > 0.99
    assert ((code == low) | (code == high))[same].all()
