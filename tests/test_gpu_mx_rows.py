"""The microscaled norm of more rows than 32-bit thread indices can count."""
import numpy as np
import pytest

import mx_reference as mx
from test_gpu_mx import ctx, release  # noqa: F401 (fixtures)
from voxelengine import cuda as cu

pytestmark = pytest.mark.gpu


def test_rmsnorm_of_2_to_27_rows(ctx):
    """Short rows have a warp each, 8 to a block: 2^27 of them are 2^32 threads. 9 GB of codes."""
    rows, cols, seen = (1 << 27) + 5, 1, 4096
    x = ctx.buffer(rows * 2).fill(0)
    out = cu.MxMatrix(ctx.buffer(cu.mx_code_bytes(mx.FP4, rows, cols)).fill(0xA5).ptr, ctx.buffer(cu.mx_scale_bytes(rows, cols)).fill(0xA5).ptr,
                      rows, cols, mx.FP4)
    codes, scales = ctx._bufs[-2], ctx._bufs[-1]
    rng = np.random.default_rng(0)
    ends = [0, rows - seen]
    # Of one value and eps 1, x / sqrt(x^2 + 1): multiples of 1/16 that are not 0, none of whose
    # norms lies within 2^-18 of a rounding boundary (asserted).
    values = [(rng.integers(1, 64, seen) * rng.choice([-1, 1], seen) / 16).astype(np.float16) for _ in ends]
    for at, v in zip(ends, values):
        x.upload(v, at * 2)
    ctx.mx_rmsnorm(cu.MxNormArgs(x=x.ptr, x_type=cu.F16, x_stride=cols, eps=1.0, out=out))
    for at, v in zip(ends, values):
        v = v.astype(np.float64)[:, None]
        y = v / np.sqrt(v * v + 1)
        code, byte = mx.quantize(y, mx.FP4)
        for f in (1 - 2.0 ** -18, 1 + 2.0 ** -18):
            assert all(np.array_equal(a, b) for a, b in zip(mx.quantize(y * f, mx.FP4), (code, byte)))
        assert np.array_equal(codes.download(np.uint8, (seen, 64), at * 64), code)
        first = at // 128 * 128
        tail = scales.download(np.uint8, cu.mx_scale_bytes(at + seen - first, cols), first // 128 * 512)
        assert np.array_equal(mx.untile(tail, at + seen - first, cols)[at - first:], byte)
    assert (codes.download(np.uint8, 64, (rows // 2) * 64) == 0).all()


def test_rmsnorm_refuses_what_it_cannot_count(ctx):
    """Sizes alone: refused before anything is launched, so no memory of that size is needed."""
    x = ctx.buffer(1024)

    def norm(rows, cols):
        ctx.mx_rmsnorm(cu.MxNormArgs(x=x.ptr, x_type=cu.F16, x_stride=1 << 32, eps=1.0, out=cu.MxMatrix(x.ptr, x.ptr, rows, cols, mx.FP8)))

    for rows, cols in [(1, 2 ** 32 - 8191), (1, 0xffffff80), (2 ** 31, 1)]:
        with pytest.raises(cu.OpureError) as e:
            norm(rows, cols)
        assert e.value.status == cu.ERR_UNSUPPORTED


def test_quantize_and_dequantize_refuse_what_they_cannot_count(ctx):
    x = ctx.buffer(1024)
    for rows, cols in [(2 ** 29 - 63, 1), (2 ** 28, 129), (2 ** 32 - 1, 1)]:
        m = cu.MxMatrix(x.ptr, x.ptr, rows, cols, mx.FP4)
        for call in (lambda: ctx.mx_quantize(x.ptr, cu.F16, 1 << 32, m), lambda: ctx.mx_dequantize(m, x.ptr, cu.F16, 1 << 32)):
            with pytest.raises(cu.OpureError) as e:
                call()
            assert e.value.status == cu.ERR_UNSUPPORTED
