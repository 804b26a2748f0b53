"""The microscaled norm of rows whose squares or their mean leave fp32's range."""
import numpy as np
import pytest

import mx_reference as mx
from test_gpu_mx import FORMATS, Mx, Rows, check_quantized, ctx, release  # noqa: F401 (fixtures)
from voxelengine import cuda as cu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("cols", [64, 640, 17000])
def test_rows_of_any_magnitude(ctx, t, fmt, cols):
    """From the last subnormals to near the largest value: a finite row has a finite norm."""
    rng = np.random.default_rng(cols)
    sizes = [3e37, 1e30, 4e19, 1e15, 1e-10, 1e-16, 1e-19, 1e-25, 1e-33, 1e-37]
    sizes += [1e-40] if t == "f32" else []
    rows = len(sizes)
    X, S = Rows(ctx, rows, cols, t), Rows(ctx, rows, cols, t)
    x = X.put(np.clip(rng.standard_normal((rows, cols)), -10, 10) * np.array(sizes)[:, None])
    gain = (1 + 0.1 * rng.standard_normal(cols)).astype(np.float16)
    out = Mx(ctx, rows, cols, fmt)
    ctx.mx_rmsnorm(cu.MxNormArgs(x=X.ptr, x_type=cu.VALUE_TYPES[t], x_stride=cols, sum=S.ptr, gain=ctx.to_device(gain).ptr, eps=0.0,
                                 out=out.m))
    assert np.array_equal(S.get(), x)
    y = x / np.sqrt((x * x).mean(1, keepdims=True)) * gain.astype(np.float64)
    # Squares are added in fp32 eight at a time, the rest in 64 bits; one product is rounded to
    # fp32 at the end: under 2^-22. A boundary lies that near a value with probability 2^-22 / 2^-5.
    check_quantized(out.get(), y, cols, fmt, 2.0 ** -22, 2.0 ** -16)


def test_rows_without_a_norm(ctx):
    """An infinity or NaN, and with eps = 0 a row of zeros: NaN where the definition has one, zeros
    where it has finite / infinite; other rows keep theirs."""
    rows, cols = 4, 96
    x = np.ones((rows, cols))
    x[0, 40], x[1, 3], x[2] = np.inf, np.nan, 0
    X, out = Rows(ctx, rows, cols, "f32"), Mx(ctx, rows, cols, mx.FP8)
    X.put(x)
    ctx.mx_rmsnorm(cu.MxNormArgs(x=X.ptr, x_type=cu.F32, x_stride=cols, eps=0.0, out=out.m))
    code, byte = out.get()
    assert (byte[0, :3] == [0, 255, 0]).all() and (code[0] == 0).all()
    assert (byte[1:3, :3] == 255).all()
    want = mx.quantize(np.ones((1, cols)), mx.FP8)
    assert np.array_equal(code[3], want[0][0]) and np.array_equal(byte[3], want[1][0])
