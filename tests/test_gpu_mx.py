"""Microscaled linear-layer kernels against a plain 64-bit implementation (mx_reference).

Quantising and dequantising are exact: every step of the definition (largest magnitude, power
of two, rounding to the grid) is exact in fp32, so bytes are compared for equality. Bounds of
the others are stated where they are derived.
"""
import numpy as np
import pytest
import torch

import mx_reference as mx
from voxelengine import cuda as cu

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f16", "bf16"]
FORMATS = [cu.MX_FP4, cu.MX_FP8]
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
HALF_ULP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half of the last subnormal, or less
GUARD = 0xA5


@pytest.fixture(scope="module")
def ctx():
    c = cu.Ctx(0)
    yield c
    c.close()


@pytest.fixture(autouse=True)
def release(ctx):
    first = len(ctx._bufs)
    yield
    assert ctx.last_error() == 0
    for b in ctx._bufs[first:]:
        b.free()
    del ctx._bufs[first:]


def encode(x, t):
    """float64 -> (bytes of the type, the values they hold in 64 bits)."""
    f = torch.from_numpy(np.asarray(x, np.float32)).to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[t])
    return f.view(torch.int32 if t == "f32" else torch.int16).numpy(), f.double().numpy()


def decode(raw, t):
    f = torch.from_numpy(np.ascontiguousarray(raw)).view({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[t])
    return f.double().numpy()


class Rows:
    """Rows of a type on the device with a stride, an offset of `shift` values, and guard bytes
    everywhere else."""

    def __init__(self, ctx, rows, cols, t, stride=None, shift=0):
        self.t, self.rows, self.cols, self.stride, self.shift = t, rows, cols, stride or cols, shift
        self.dtype = np.int32 if t == "f32" else np.int16
        self.n = shift + rows * self.stride + 16
        self.buf = ctx.buffer(self.n * SIZE[t]).fill(GUARD)
        self.ptr = self.buf.ptr + shift * SIZE[t]

    def _all(self):
        a = self.buf.download(self.dtype, self.n)
        return a, a[self.shift:self.shift + self.rows * self.stride].reshape(self.rows, self.stride)

    def put(self, x):
        raw, held = encode(x, self.t)
        a, body = self._all()
        body[:, :self.cols] = raw
        self.buf.upload(a)
        return held

    def get(self):
        a, body = self._all()
        got = decode(body[:, :self.cols].copy(), self.t)
        body[:, :self.cols] = np.frombuffer(bytes([GUARD] * SIZE[self.t]), self.dtype)[0]
        assert (a.view(np.uint8) == GUARD).all(), "wrote outside its rows"
        return got


class Mx:
    """A microscaled matrix on the device; bytes that a kernel has no business in hold GUARD."""

    def __init__(self, ctx, rows, cols, fmt, code=None, byte=None, fill=GUARD):
        self.rows, self.cols, self.fmt = rows, cols, fmt
        self.nc, self.ns = cu.mx_code_bytes(fmt, rows, cols), cu.mx_scale_bytes(rows, cols)
        self.c, self.s = ctx.buffer(self.nc + 64).fill(GUARD), ctx.buffer(self.ns + 64).fill(GUARD)
        if code is not None:
            self.c.upload(code)
            self.s.upload(mx.tiles(byte, cols, fill))
        self.m = cu.MxMatrix(self.c.ptr, self.s.ptr, rows, cols, fmt)

    def get(self):
        """(codes, scale bytes), having checked that nothing else was written."""
        c, s = self.c.download(np.uint8, self.nc + 64), self.s.download(np.uint8, self.ns + 64)
        assert (c[self.nc:] == GUARD).all()
        byte = mx.untile(s, self.rows, self.cols)
        s[mx.scale_offsets(self.rows, self.cols)] = GUARD
        assert (s == GUARD).all(), "wrote scales of rows that are not there"
        return c[:self.nc].reshape(self.rows, -1), byte


def random_mx(ctx, rng, rows, cols, fmt, std=1.0, fill=GUARD):
    x = rng.standard_normal((rows, cols)) * std
    x *= np.exp2(rng.integers(-3, 4, cols))
    code, byte = mx.quantize(x, fmt)
    return Mx(ctx, rows, cols, fmt, code, byte, fill), mx.values(code, byte, cols, fmt)


# ---- quantise ----------------------------------------------------------------------------
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,cols,stride,shift", [
    (1, 1, None, 0), (1, 31, None, 0), (3, 32, None, 0), (2, 33, 40, 0), (127, 127, None, 0), (128, 128, None, 0),
    (129, 129, 136, 0), (5, 576, None, 0), (5, 576, 577, 0), (4, 576, None, 1), (33, 1100, 1104, 8), (300, 2048, None, 0),
    (2, 16392, None, 0)])
def test_quantize(ctx, t, fmt, rows, cols, stride, shift):
    rng = np.random.default_rng(rows * 1000 + cols)
    src = Rows(ctx, rows, cols, t, stride, shift)
    x = src.put(rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-8, 8, (rows, 1))))
    out = Mx(ctx, rows, cols, fmt)
    ctx.mx_quantize(src.ptr, cu.VALUE_TYPES[t], src.stride, out.m)
    code, byte = out.get()
    want_code, want_byte = mx.quantize(x, fmt)
    assert np.array_equal(byte, want_byte)
    assert np.array_equal(code, want_code)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shift", range(8))
def test_quantize_and_back_from_any_address(ctx, t, shift):
    """Every offset from a 16-byte boundary that a 2-byte type can have, and rows that end anywhere."""
    rng = np.random.default_rng(shift)
    for rows, cols, stride in [(3, 1100 + shift, None), (9, 16, 17), (5, 145, 149), (2, 15, None)]:
        src, y, out = Rows(ctx, rows, cols, t, stride, shift), Rows(ctx, rows, cols, t, stride, shift), Mx(ctx, rows, cols, mx.FP8)
        x = src.put(rng.standard_normal((rows, cols)))
        ctx.mx_quantize(src.ptr, cu.VALUE_TYPES[t], src.stride, out.m)
        code, byte = out.get()
        want_code, want_byte = mx.quantize(x, mx.FP8)
        assert np.array_equal(byte, want_byte) and np.array_equal(code, want_code)
        ctx.mx_dequantize(out.m, y.ptr, cu.VALUE_TYPES[t], y.stride)
        assert np.array_equal(y.get(), encode(mx.values(want_code, want_byte, cols, mx.FP8), t)[1])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_and_back_many_unaligned_rows(ctx, t, fmt):
    rng = np.random.default_rng(7)
    rows, cols = 3001, 1611
    src, y, out = Rows(ctx, rows, cols, t, None, 1), Rows(ctx, rows, cols, t, 1613, 3), Mx(ctx, rows, cols, fmt)
    x = src.put(rng.standard_normal((rows, cols)))
    ctx.mx_quantize(src.ptr, cu.VALUE_TYPES[t], src.stride, out.m)
    code, byte = out.get()
    want_code, want_byte = mx.quantize(x, fmt)
    assert np.array_equal(byte, want_byte) and np.array_equal(code, want_code)
    ctx.mx_dequantize(out.m, y.ptr, cu.VALUE_TYPES[t], y.stride)
    assert np.array_equal(y.get(), encode(mx.values(want_code, want_byte, cols, fmt), t)[1])


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_special_values(ctx, fmt):
    """Empty blocks, ties, the limits of fp32, subnormals, infinities and NaN, one per block."""
    g = mx.GRID[fmt]
    ties = ((g[1:] + g[:-1]) / 2)[:24]
    rows = np.zeros((16, 64), np.float64)
    rows[1, :24] = np.resize(ties, 24)
    rows[1, 31] = g[-1]
    rows[2] = -rows[1]
    rows[3, :3] = [3.4028234663852886e38, -1e38, 1.0]
    rows[4, :3] = [2.0 ** -149, 2.0 ** -130, -2.0 ** -127]
    rows[5, :3] = [2.0 ** -126, 2.0 ** -125 * 1.5, 0]
    rows[6, 5] = np.inf
    rows[7, 40] = -np.inf
    rows[8, 63] = np.nan
    rows[9, 0] = np.nextafter(np.float32(8), np.float32(0))
    rows[10, :2] = [-0.0, 0.0]
    rows[11, :2] = [2.0 ** 120, 2.0 ** -120]
    rows[12] = g[-1] * 1.2
    src = Rows(ctx, 16, 64, "f32")
    x = src.put(rows)
    out = Mx(ctx, 16, 64, fmt)
    ctx.mx_quantize(src.ptr, cu.F32, 64, out.m)
    code, byte = out.get()
    want_code, want_byte = mx.quantize(x, fmt)
    assert np.array_equal(byte, want_byte)
    assert np.array_equal(mx.values(code, byte, 64, fmt), mx.values(want_code, want_byte, 64, fmt), equal_nan=True)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,cols,stride,shift", [(1, 1, None, 0), (130, 300, 307, 3), (7, 129, 136, 8), (256, 2048, None, 0)])
def test_dequantize(ctx, t, fmt, rows, cols, stride, shift):
    rng = np.random.default_rng(cols)
    src, want = random_mx(ctx, rng, rows, cols, fmt)
    y = Rows(ctx, rows, cols, t, stride, shift)
    ctx.mx_dequantize(src.m, y.ptr, cu.VALUE_TYPES[t], y.stride)
    got = y.get()
    assert np.array_equal(got, encode(want, t)[1])


@pytest.mark.parametrize("fmt", FORMATS)
def test_dequantize_every_code_and_scale(ctx, fmt):
    n = 16 if fmt == cu.MX_FP4 else 256
    code = np.resize(np.arange(n, dtype=np.uint8), (256, 256))
    byte = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 8, 1)
    packed = code if fmt == cu.MX_FP8 else code[:, ::2] | (code[:, 1::2] << 4)
    src = Mx(ctx, 256, 256, fmt, packed, byte)
    y = Rows(ctx, 256, 256, "f32")
    ctx.mx_dequantize(src.m, y.ptr, cu.F32, 256)
    with np.errstate(over="ignore"):
        want = mx.values(packed, byte, 256, fmt).astype(np.float32).astype(np.float64)
    assert np.array_equal(y.get(), want, equal_nan=True)


# ---- norm --------------------------------------------------------------------------------
def check_quantized(got, y, cols, fmt, rel, most_flips):
    """A result computed in fp32 with relative error `rel`, then quantised: every value is
    within half a step of its code (or beyond the limit), and at most a share `most_flips` of
    codes differ from those of the exact result (values within `rel` of a rounding boundary)."""
    code, byte = got
    want_code, want_byte = mx.quantize(y, fmt)
    v = mx.values(code, byte, cols, fmt)
    # Half a step: 2^-4 (E4M3) or 2^-2 (E2M1) of the value, or of the last subnormal; a value
    # above the limit (up to 512 or 8 at the block's scale) is off by its distance to it.
    step, small, over = (2.0 ** -4, 2.0 ** -10, 64.0) if fmt == cu.MX_FP8 else (2.0 ** -2, 2.0 ** -2, 2.0)
    s = np.repeat(np.exp2(byte.astype(np.float64) - 127), 32, 1)[:, :cols]
    top = mx.GRID[fmt][-1] * s
    bound = np.maximum(np.abs(y) * step, small * s) * (1 + 16 * rel) + np.where(np.abs(y) > top, over * s, 0)
    assert (np.abs(v - y) <= bound).all()
    flips = np.mean(code != want_code)
    assert flips <= most_flips + 2.0 / code.size, flips
    assert np.mean(byte != want_byte) <= most_flips + 1.0 / byte.size


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,cols,stride,shift", [
    (1, 1, None, 0), (1, 576, None, 0), (3, 33, 48, 0), (130, 577, None, 0), (64, 2048, None, 0), (5, 2048, 2056, 1),
    (2, 4104, None, 0), (3, 8192, None, 0), (2, 16385, 16392, 0), (2, 20000, None, 0), (1300, 64, None, 0), (1201, 300, 304, 8),
    (1211, 75, None, 0), (1190, 512, 513, 1), (3, 9001, None, 0), (2, 17001, 17003, 1)])
def test_rmsnorm(ctx, t, fmt, rows, cols, stride, shift):
    rng = np.random.default_rng(cols + rows)
    X, R, S = (Rows(ctx, rows, cols, t, stride, shift) for _ in range(3))
    x, r = X.put(rng.standard_normal((rows, cols))), R.put(rng.standard_normal((rows, cols)) * 3)
    gain, g = encode(1 + 0.1 * rng.standard_normal(cols), "f16")
    out = Mx(ctx, rows, cols, fmt)
    ctx.mx_rmsnorm(cu.MxNormArgs(X.ptr, cu.VALUE_TYPES[t], X.stride, R.ptr, S.ptr, ctx.to_device(gain).ptr, 1e-5, out.m))
    s = x + r
    # One fp32 addition, then rounding to the type.
    assert (np.abs(S.get() - s) <= np.abs(s) * (2.0 ** -24 + HALF_ULP[t]) * 1.001 + TINY[t]).all()
    y = s / np.sqrt((s * s).mean(1, keepdims=True) + 1e-5) * g
    # fp32: the sum of squares over cols terms, a root, a division, three products: under 2^-18
    # for these cols (partial sums of at most 128 terms a thread, then a tree). A boundary lies
    # within 2^-18 of a value with probability 2^-18 / 2^-4 x 2 at most.
    check_quantized(out.get(), y, cols, fmt, 2.0 ** -18, 2.0 ** -12)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shift", range(8))
def test_rmsnorm_in_place_at_any_address(ctx, t, shift):
    """x and the residual at different offsets from a 16-byte boundary, the sum over either: values
    that share a word with other lanes' or rows' stay what they are."""
    rng = np.random.default_rng(shift)
    for rows, cols, stride in [(5, 1100 + shift, None), (3, 8, 9), (4, 145, 149), (1200, 75, None), (2, 9001, None), (2, 17001, None)]:
        X, R = Rows(ctx, rows, cols, t, stride, shift), Rows(ctx, rows, cols, t, stride, (shift * 3 + 1) % 8)
        x, r = X.put(rng.standard_normal((rows, cols))), R.put(rng.standard_normal((rows, cols)))
        S, other, kept = (X, R, r) if shift % 2 else (R, X, x)
        out = Mx(ctx, rows, cols, mx.FP8)
        ctx.mx_rmsnorm(cu.MxNormArgs(x=X.ptr, x_type=cu.VALUE_TYPES[t], x_stride=X.stride, residual=R.ptr, sum=S.ptr, eps=1e-5, out=out.m))
        s = x + r
        assert (np.abs(S.get() - s) <= np.abs(s) * (2.0 ** -24 + HALF_ULP[t]) * 1.001 + TINY[t]).all()
        assert np.array_equal(other.get(), kept)
        check_quantized(out.get(), s / np.sqrt((s * s).mean(1, keepdims=True) + 1e-5), cols, mx.FP8, 2.0 ** -18, 2.0 ** -12)


@pytest.mark.parametrize("t,rows,cols,stride", [
    ("f16", 2500, 1024, None), ("bf16", 2501, 1001, None), ("f16", 330, 7524, None), ("bf16", 160, 16384, None), ("f16", 161, 16000, 16003)])
def test_rmsnorm_more_octets_than_threads(ctx, t, rows, cols, stride):
    rng = np.random.default_rng(rows)
    X, R = Rows(ctx, rows, cols, t, stride), Rows(ctx, rows, cols, t, stride)
    x, r = X.put(rng.standard_normal((rows, cols))), R.put(rng.standard_normal((rows, cols)))
    out = Mx(ctx, rows, cols, mx.FP8)
    ctx.mx_rmsnorm(cu.MxNormArgs(x=X.ptr, x_type=cu.VALUE_TYPES[t], x_stride=X.stride, residual=R.ptr, sum=X.ptr, eps=1e-5, out=out.m))
    s = x + r
    assert (np.abs(X.get() - s) <= np.abs(s) * (2.0 ** -24 + HALF_ULP[t]) * 1.001 + TINY[t]).all()
    check_quantized(out.get(), s / np.sqrt((s * s).mean(1, keepdims=True) + 1e-5), cols, mx.FP8, 2.0 ** -18, 2.0 ** -12)


def test_rmsnorm_of_values_whose_squares_fp32_cannot_hold(ctx):
    """Sums of 8 squares that overflow, and squares near the last subnormal; the mean is a float."""
    rng = np.random.default_rng(3)
    rows, cols = 2, 640
    X = Rows(ctx, rows, cols, "f32")
    x = X.put(rng.standard_normal((rows, cols)) * np.array([[1e19], [1e-17]]))
    out = Mx(ctx, rows, cols, mx.FP8)
    ctx.mx_rmsnorm(cu.MxNormArgs(x=X.ptr, x_type=cu.F32, x_stride=cols, eps=0.0, out=out.m))
    check_quantized(out.get(), x / np.sqrt((x * x).mean(1, keepdims=True)), cols, mx.FP8, 2.0 ** -18, 2.0 ** -12)


def test_rmsnorm_options(ctx):
    """No residual, no gain, no sum; sum over x; sum over the residual; a zero row; a NaN row."""
    rng = np.random.default_rng(5)
    rows, cols = 4, 600
    base, res = rng.standard_normal((rows, cols)), rng.standard_normal((rows, cols))
    base[1], res[1] = 0, 0
    base[2, 7] = np.nan
    ok = [0, 1, 3]
    for which in ("plain", "over x", "over residual"):
        X, R = Rows(ctx, rows, cols, "f32"), Rows(ctx, rows, cols, "f32")
        x, r = X.put(base), R.put(res)
        out = Mx(ctx, rows, cols, cu.MX_FP8)
        a = cu.MxNormArgs(x=X.ptr, x_type=cu.F32, x_stride=cols, eps=1e-5, out=out.m)
        if which != "plain":
            a.residual, a.sum = R.ptr, X.ptr if which == "over x" else R.ptr
        ctx.mx_rmsnorm(a)
        s = x if which == "plain" else x + r
        code, byte = out.get()
        assert (byte[2] == 255).all() or (byte[2, :19] == 255).all()
        assert (byte[1] == 0).all() and (code[1] == 0).all()
        y = s / np.sqrt((s * s).mean(1, keepdims=True) + 1e-5)
        check_quantized((code[ok], byte[ok]), y[ok], cols, cu.MX_FP8, 2.0 ** -18, 2.0 ** -12)
        got = X.get() if which == "over x" else R.get()
        if which != "plain":
            assert np.allclose(got[ok], s[ok], rtol=2.0 ** -23, atol=0)
        else:
            assert np.array_equal(got, r)


# ---- product -----------------------------------------------------------------------------
def product_bound(x, w, y, t):
    """fp32 sums of exact products in any order, each addition off by at most 2^-22 of the
    magnitudes summed (tensor-core additions may truncate): blocks of 32 are added one after
    another, up to 8 pieces of K are joined, and the scales multiply exactly; then one rounding
    to the type."""
    mag = np.abs(x) @ np.abs(w).T
    return (x.shape[1] / 32 + 16) * 2.0 ** -22 * mag + np.abs(y) * HALF_ULP[t] * 1.001 + TINY[t]


SHAPES = [  # n, rows, cols
    (1, 1, 1), (1, 32, 32), (1, 576, 576), (2, 33, 96), (3, 130, 129), (5, 1003, 1100), (8, 960, 576), (9, 257, 640),
    (16, 128, 128), (17, 576, 1536), (33, 300, 64), (64, 576, 576), (65, 129, 2048), (127, 200, 320), (128, 256, 256),
    (129, 384, 1000), (200, 1536, 576), (256, 513, 130), (300, 770, 388), (1, 2048, 8192), (4, 49152, 576), (513, 1025, 448)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n,rows,cols", SHAPES)
def test_gemm_store(ctx, fmt, n, rows, cols):
    rng = np.random.default_rng(n * 7 + rows + cols)
    X, x = random_mx(ctx, rng, n, cols, fmt)
    W, w = random_mx(ctx, rng, rows, cols, cu.MX_FP4, 0.02)
    y = x @ w.T
    for t in TYPES:
        Y = Rows(ctx, n, rows, t)
        ctx.mx_gemm(cu.MxGemmArgs(w=W.m, x=X.m, y=Y.ptr, y_type=cu.VALUE_TYPES[t], y_stride=rows))
        assert (np.abs(Y.get() - y) <= product_bound(x, w, y, t)).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n,rows,cols,stride,shift", [
    (1, 576, 1536, None, 0), (7, 100, 200, 104, 0), (40, 576, 576, 577, 1), (130, 300, 260, 304, 8), (300, 640, 512, None, 0),
    (260, 1000, 384, 1003, 3)])
def test_gemm_add(ctx, t, fmt, n, rows, cols, stride, shift):
    rng = np.random.default_rng(n + rows)
    X, x = random_mx(ctx, rng, n, cols, fmt)
    W, w = random_mx(ctx, rng, rows, cols, cu.MX_FP4, 0.02)
    for in_place in (False, True):
        R, Y = Rows(ctx, n, rows, t, stride, shift), Rows(ctx, n, rows, t, stride, shift)
        r = R.put(rng.standard_normal((n, rows)))
        if in_place:
            Y = R
        ctx.mx_gemm(cu.MxGemmArgs(w=W.m, x=X.m, epilogue=cu.EPI_ADD, y=Y.ptr, y_type=cu.VALUE_TYPES[t], y_stride=Y.stride,
                                  residual=R.ptr))
        y = x @ w.T + r
        bound = product_bound(x, w, y, t) + 2.0 ** -23 * (np.abs(r) + np.abs(y))
        assert (np.abs(Y.get() - y) <= bound).all()
        if not in_place:
            assert np.array_equal(R.get(), r)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("out_fmt", FORMATS)
@pytest.mark.parametrize("n,ff,cols", [
    (1, 1, 32), (1, 1536, 576), (3, 33, 100), (16, 160, 256), (64, 1536, 576), (70, 100, 300), (129, 128, 128),
    (140, 333, 576), (300, 512, 260), (260, 1536, 576)])
def test_gemm_swiglu(ctx, fmt, out_fmt, n, ff, cols):
    rng = np.random.default_rng(n + ff)
    X, x = random_mx(ctx, rng, n, cols, fmt, 0.5)
    W, w = random_mx(ctx, rng, 2 * ff, cols, cu.MX_FP4, 0.05)
    out = Mx(ctx, n, ff, out_fmt)
    ctx.mx_gemm(cu.MxGemmArgs(w=W.m, x=X.m, epilogue=cu.EPI_SWIGLU, out=out.m))
    g, u = x @ w[:ff].T, x @ w[ff:].T
    y = g / (1 + np.exp(-g)) * u
    code, byte = out.get()
    want_code, want_byte = mx.quantize(y, out_fmt)
    # The product's error, carried through silu (slope at most 1.1) and the multiplication,
    # against the step of each value: few codes may differ, each by a neighbour.
    err = 1.1 * product_bound(x, w[:ff], g, "f32") * np.abs(u) + 1.1 * product_bound(x, w[ff:], u, "f32") * np.abs(g)
    s = np.repeat(np.exp2(byte.astype(np.float64) - 127), 32, 1)[:, :ff]
    half, small, over = (2.0 ** -4, 2.0 ** -10, 64.0) if out_fmt == cu.MX_FP8 else (2.0 ** -2, 2.0 ** -2, 2.0)
    v = mx.values(code, byte, ff, out_fmt)
    bound = np.maximum(np.abs(y) * half, small * s) * (1 + 2.0 ** -20) + 2 * err
    bound += np.where(np.abs(y) + err > mx.GRID[out_fmt][-1] * s, over * s, 0)
    assert (np.abs(v - y) <= bound).all()
    assert np.mean(code != want_code) <= 2e-3 + 2.0 / code.size
    assert np.mean(byte != want_byte) <= 2e-3 + 1.0 / byte.size


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n,rows,cols,stride,shift", [
    (2, 100, 200, 103, 1), (40, 300, 260, 304, 8), (64, 129, 1000, 131, 1), (300, 1000, 384, 1008, 0), (300, 1003, 384, 1008, 8),
    (260, 1001, 130, 1003, 3)])
def test_gemm_store_strided(ctx, t, fmt, n, rows, cols, stride, shift):
    """Rows with room between them, which stays as it was, at every alignment."""
    rng = np.random.default_rng(n + rows + cols)
    X, x = random_mx(ctx, rng, n, cols, fmt)
    W, w = random_mx(ctx, rng, rows, cols, cu.MX_FP4, 0.02)
    y = x @ w.T
    Y = Rows(ctx, n, rows, t, stride, shift)
    ctx.mx_gemm(cu.MxGemmArgs(w=W.m, x=X.m, y=Y.ptr, y_type=cu.VALUE_TYPES[t], y_stride=stride))
    assert (np.abs(Y.get() - y) <= product_bound(x, w, y, t)).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("epi,t", [(cu.EPI_STORE, "f32"), (cu.EPI_STORE, "bf16"), (cu.EPI_ADD, "f32"), (cu.EPI_ADD, "f16"),
                                   (cu.EPI_SWIGLU, "f32")])
def test_gemm_many_tiles(ctx, fmt, epi, t):
    """More 256 x 256 tiles than pairs of SMs, so that a pair goes from one accumulator to the other
    and back, with an end inside the last tiles."""
    rng = np.random.default_rng(6)
    n, rows, cols = 2000, 5100 if epi == cu.EPI_SWIGLU else 5000, 640
    X, x = random_mx(ctx, rng, n, cols, fmt)
    W, w = random_mx(ctx, rng, rows, cols, cu.MX_FP4, 0.02)
    y = x @ w.T
    if epi == cu.EPI_SWIGLU:
        out = Mx(ctx, n, rows // 2, cu.MX_FP8)
        ctx.mx_gemm(cu.MxGemmArgs(w=W.m, x=X.m, epilogue=epi, out=out.m))
        g, u = y[:, :rows // 2], y[:, rows // 2:]
        want = g / (1 + np.exp(-g)) * u
        code, byte = out.get()
        v = mx.values(code, byte, rows // 2, cu.MX_FP8)
        s = np.repeat(np.exp2(byte.astype(np.float64) - 127), 32, 1)[:, :rows // 2]
        # Half a step of E4M3, the product's error as in test_gemm_swiglu, and the limit of 448.
        err = 1.1 * product_bound(x, w[:rows // 2], g, "f32") * np.abs(u) + 1.1 * product_bound(x, w[rows // 2:], u, "f32") * np.abs(g)
        bound = np.maximum(np.abs(want) * 2.0 ** -4, 2.0 ** -10 * s) * (1 + 2.0 ** -20) + 2 * err
        assert (np.abs(v - want) <= bound + np.where(np.abs(want) + err > 448 * s, 64 * s, 0)).all()
        assert np.mean(code != mx.quantize(want, cu.MX_FP8)[0]) <= 2e-3
        return
    Y, R = Rows(ctx, n, rows, t), Rows(ctx, n, rows, t)
    a = cu.MxGemmArgs(w=W.m, x=X.m, epilogue=epi, y=Y.ptr, y_type=cu.VALUE_TYPES[t], y_stride=rows)
    if epi == cu.EPI_ADD:
        r = R.put(rng.standard_normal((n, rows)))
        a.residual = R.ptr
        y = y + r
    ctx.mx_gemm(a)
    assert (np.abs(Y.get() - y) <= product_bound(x, w, y, t) + 2.0 ** -22 * np.abs(y)).all()


@pytest.mark.parametrize("n,rows,cols", [(1, 130, 576), (20, 200, 300), (300, 520, 300)])
def test_gemm_nan_stays_in_its_row_and_column(ctx, n, rows, cols):
    """A NaN block of one token and of one weight row; scales of rows that are not there are NaN too."""
    rng = np.random.default_rng(3)
    x, w = rng.standard_normal((n, cols)), rng.standard_normal((rows, cols))
    i, r = n - 1, rows // 2
    x[i, 40], w[r, cols - 1] = np.inf, np.nan
    xc, xb = mx.quantize(x, cu.MX_FP8)
    wc, wb = mx.quantize(w, cu.MX_FP4)
    X, W = Mx(ctx, n, cols, cu.MX_FP8, xc, xb, fill=255), Mx(ctx, rows, cols, cu.MX_FP4, wc, wb, fill=255)
    Y = Rows(ctx, n, rows, "f32")
    ctx.mx_gemm(cu.MxGemmArgs(w=W.m, x=X.m, y=Y.ptr, y_type=cu.F32, y_stride=rows))
    got = Y.get()
    nan = np.zeros((n, rows), bool)
    nan[i], nan[:, r] = True, True
    assert np.array_equal(np.isnan(got), nan)
    xv, wv = mx.values(xc, xb, cols, cu.MX_FP8), mx.values(wc, wb, cols, cu.MX_FP4)
    keep_i, keep_r = [k for k in range(n) if k != i], [k for k in range(rows) if k != r]
    if keep_i:
        xk, wk = xv[keep_i], wv[keep_r]
        assert (np.abs(got[np.ix_(keep_i, keep_r)] - xk @ wk.T) <= product_bound(xk, wk, xk @ wk.T, "f32")).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_gemm_extreme_scales(ctx, fmt):
    """Blocks whose scales are far apart: each row has its own power of two, from 2^-100 to 2^100."""
    rng = np.random.default_rng(8)
    n, rows, cols = 24, 96, 256
    x = rng.standard_normal((n, cols)) * np.exp2(np.linspace(-50, 50, n))[:, None]
    w = rng.standard_normal((rows, cols)) * np.exp2(np.linspace(-50, 50, rows))[:, None]
    (xc, xb), (wc, wb) = mx.quantize(x, fmt), mx.quantize(w, cu.MX_FP4)
    X, W = Mx(ctx, n, cols, fmt, xc, xb), Mx(ctx, rows, cols, cu.MX_FP4, wc, wb)
    Y = Rows(ctx, n, rows, "f32")
    ctx.mx_gemm(cu.MxGemmArgs(w=W.m, x=X.m, y=Y.ptr, y_type=cu.F32, y_stride=rows))
    xv, wv = mx.values(xc, xb, cols, fmt), mx.values(wc, wb, cols, cu.MX_FP4)
    want = xv @ wv.T
    assert (np.abs(Y.get() - want) <= product_bound(xv, wv, want, "f32")).all()


@pytest.mark.parametrize("n,rows,cols,epi", [(1, 2048, 8192, 0), (64, 576, 1536, 0), (300, 1024, 576, 0), (64, 1536, 576, 2),
                                             (300, 1536, 576, 2)])
def test_gemm_same_bits_every_time(ctx, n, rows, cols, epi):
    rng = np.random.default_rng(2)
    X, _ = random_mx(ctx, rng, n, cols, cu.MX_FP8)
    W, _ = random_mx(ctx, rng, rows, cols, cu.MX_FP4, 0.02)
    got = []
    for _ in range(3):
        if epi == cu.EPI_SWIGLU:
            out = Mx(ctx, n, rows // 2, cu.MX_FP8)
            ctx.mx_gemm(cu.MxGemmArgs(w=W.m, x=X.m, epilogue=epi, out=out.m))
            got.append(np.concatenate([a.ravel() for a in out.get()]))
        else:
            Y = Rows(ctx, n, rows, "f32")
            ctx.mx_gemm(cu.MxGemmArgs(w=W.m, x=X.m, y=Y.ptr, y_type=cu.F32, y_stride=rows))
            got.append(Y.get())
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])


def test_calls_in_a_graph_and_back_to_back(ctx):
    """norm -> SwiGLU product -> product as one captured graph equals the calls one by one."""
    rng = np.random.default_rng(4)
    n, d, ff = 20, 576, 1536
    X = Rows(ctx, n, d, "f32")
    X.put(rng.standard_normal((n, d)))
    W1, _ = random_mx(ctx, rng, 2 * ff, d, cu.MX_FP4, 0.02)
    W2, _ = random_mx(ctx, rng, d, ff, cu.MX_FP4, 0.02)

    def layer(Y):
        a, h = Mx(ctx, n, d, cu.MX_FP8), Mx(ctx, n, ff, cu.MX_FP8)
        ctx.sync()

        def go():
            ctx.mx_rmsnorm(cu.MxNormArgs(x=X.ptr, x_type=cu.F32, x_stride=d, eps=1e-5, out=a.m))
            ctx.mx_gemm(cu.MxGemmArgs(w=W1.m, x=a.m, epilogue=cu.EPI_SWIGLU, out=h.m))
            ctx.mx_gemm(cu.MxGemmArgs(w=W2.m, x=h.m, epilogue=cu.EPI_ADD, y=Y.ptr, y_type=cu.F32, y_stride=d, residual=X.ptr))
        return go

    Y1, Y2 = Rows(ctx, n, d, "f32"), Rows(ctx, n, d, "f32")
    layer(Y1)()
    one = Y1.get()
    go = layer(Y2)
    with cu.Graph(ctx) as g:
        go()
    for _ in range(3):
        g.launch()
    assert np.array_equal(Y2.get(), one)
    g.free()


def test_calls_allocate_nothing(ctx):
    rng = np.random.default_rng(1)
    n, d, ff = 150, 576, 1500
    X, Y = Rows(ctx, n, d, "f32"), Rows(ctx, n, d, "f32")
    X.put(rng.standard_normal((n, d)))
    W1, _ = random_mx(ctx, rng, 2 * ff, d, cu.MX_FP4, 0.02)
    W2, _ = random_mx(ctx, rng, d, ff, cu.MX_FP4, 0.02)
    a, h = Mx(ctx, n, d, cu.MX_FP8), Mx(ctx, n, ff, cu.MX_FP8)

    def layer():
        for rows in (1, 20, n):
            for m in (a.m, h.m):
                m.rows = rows
            ctx.mx_quantize(X.ptr, cu.F32, d, a.m)
            ctx.mx_rmsnorm(cu.MxNormArgs(x=X.ptr, x_type=cu.F32, x_stride=d, eps=1e-5, out=a.m))
            ctx.mx_gemm(cu.MxGemmArgs(w=W1.m, x=a.m, epilogue=cu.EPI_SWIGLU, out=h.m))
            ctx.mx_gemm(cu.MxGemmArgs(w=W2.m, x=h.m, y=Y.ptr, y_type=cu.F32, y_stride=d))
            ctx.mx_dequantize(a.m, Y.ptr, cu.F32, d)

    layer()
    ctx.sync()
    free = torch.cuda.mem_get_info()[0]
    for _ in range(5):
        layer()
    ctx.sync()
    assert torch.cuda.mem_get_info()[0] == free


# ---- nothing to do, and refusals -------------------------------------------------------------
def test_empty(ctx):
    e4, e8 = cu.MxMatrix(0, 0, 0, 64, cu.MX_FP4), cu.MxMatrix(0, 0, 0, 64, cu.MX_FP8)
    W, _ = random_mx(ctx, np.random.default_rng(0), 32, 64, cu.MX_FP4)
    ctx.mx_quantize(0, cu.F32, 64, e4)
    ctx.mx_dequantize(e8, 0, cu.F16, 64)
    ctx.mx_rmsnorm(cu.MxNormArgs(x_type=cu.F32, x_stride=64, out=e8))
    ctx.mx_gemm(cu.MxGemmArgs(w=W.m, x=e8, y_type=cu.F32, y_stride=32))
    ctx.sync()


def refused(status, f, *args):
    with pytest.raises(cu.OpureError) as e:
        f(*args)
    assert e.value.status == status


def test_refusals(ctx):
    rng = np.random.default_rng(0)
    X, _ = random_mx(ctx, rng, 4, 64, cu.MX_FP8)
    W, _ = random_mx(ctx, rng, 32, 64, cu.MX_FP4)
    R = Rows(ctx, 4, 64, "f32")
    bad = cu.ERR_INVALID_ARG

    def m(base, **kw):
        v = cu.MxMatrix(base.codes, base.scales, base.rows, base.cols, base.format)
        for k, x in kw.items():
            setattr(v, k, x)
        return v

    for q in (m(X.m, format=5), m(X.m, cols=0), m(X.m, codes=None), m(X.m, scales=None), m(X.m, codes=X.m.codes + 16),
              m(X.m, scales=X.m.scales + 8)):
        refused(bad, ctx.mx_quantize, R.ptr, cu.F32, 64, q)
        refused(bad, ctx.mx_dequantize, q, R.ptr, cu.F32, 64)
        refused(bad, ctx.mx_rmsnorm, cu.MxNormArgs(x=R.ptr, x_type=cu.F32, x_stride=64, eps=1e-5, out=q))
        refused(bad, ctx.mx_gemm, cu.MxGemmArgs(w=W.m, x=q, y=R.ptr, y_type=cu.F32, y_stride=32))
    refused(bad, ctx.mx_quantize, R.ptr, 3, 64, X.m)
    refused(bad, ctx.mx_quantize, R.ptr, cu.F32, 63, X.m)
    refused(bad, ctx.mx_quantize, R.ptr + 2, cu.F32, 64, X.m)
    refused(bad, ctx.mx_quantize, 0, cu.F32, 64, X.m)
    refused(bad, ctx.mx_dequantize, X.m, 0, cu.F32, 64)
    refused(bad, ctx.mx_dequantize, X.m, R.ptr, cu.F32, 60)
    refused(bad, ctx.mx_rmsnorm, cu.MxNormArgs(x=0, x_type=cu.F32, x_stride=64, out=X.m))
    refused(bad, ctx.mx_rmsnorm, cu.MxNormArgs(x=R.ptr, x_type=cu.F32, x_stride=64, gain=R.ptr + 1, out=X.m))
    refused(bad, ctx.mx_rmsnorm, cu.MxNormArgs(x=R.ptr, x_type=cu.F32, x_stride=64, sum=R.ptr + 1, out=X.m))

    def gemm(**kw):
        a = dict(w=W.m, x=X.m, y=R.ptr, y_type=cu.F32, y_stride=32)
        a.update(kw)
        return cu.MxGemmArgs(**a)

    refused(bad, ctx.mx_gemm, gemm(y=0))
    refused(bad, ctx.mx_gemm, gemm(y_stride=31))
    refused(bad, ctx.mx_gemm, gemm(y_type=7))
    refused(bad, ctx.mx_gemm, gemm(epilogue=9))
    refused(bad, ctx.mx_gemm, gemm(epilogue=cu.EPI_ADD))
    refused(bad, ctx.mx_gemm, gemm(w=m(W.m, cols=32)))
    refused(bad, ctx.mx_gemm, gemm(epilogue=cu.EPI_SWIGLU))
    refused(bad, ctx.mx_gemm, gemm(epilogue=cu.EPI_SWIGLU, out=m(X.m, cols=17)))
    refused(bad, ctx.mx_gemm, gemm(epilogue=cu.EPI_SWIGLU, w=m(W.m, rows=31), out=m(X.m, cols=15)))
    refused(cu.ERR_UNSUPPORTED, ctx.mx_gemm, gemm(w=m(X.m, rows=4)))
    refused(cu.ERR_UNSUPPORTED, ctx.mx_gemm, gemm(epilogue=cu.EPI_ARGMAX))
    ctx.call("opure_debug_inject_failure", 0, 1)
    refused(cu.ERR_INJECTED, ctx.mx_quantize, R.ptr, cu.F32, 64, X.m)
