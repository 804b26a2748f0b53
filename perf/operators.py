"""Microscaled (MX) linear-layer operators: the calls that are measured, and their plain forms.

A matrix in MX form is `codes` and `scales`: every 32 neighbouring values of a row share one
power of two. Codes are row-major with rows padded by zeros to a multiple of 128 columns; an
E4M3 (8-bit) value takes a byte, two E2M1 (4-bit) values share one, the even column in the low
half. Scales are bytes (exponent + 127) in tiles of 128 rows x 4 blocks, 512 bytes each: tile
(r / 128, k / 128), byte (r % 32) * 16 + (r / 32 % 4) * 4 + (k / 32 % 4).

Three operators, over the linear layers of the two model shapes that this framework serves
(hidden 576 / feed-forward 1536 and hidden 2048 / feed-forward 8192, vocabulary 49152):

  quantise  x -> MX. 8-bit results come back as codes and scales, 4-bit ones as the values
            that they stand for (one more call, the inverse operator).
  norm      s = x + residual; s / rms(s) * gain -> MX in 8 bits; s and the MX matrix come back.
  product   y = x W^T from an MX activation matrix (8 or 4 bits) and a 4-bit MX weight matrix,
            optionally plus a residual, or as SwiGLU of the two halves of W with an MX result.
"""
import math

import torch

own = False

FP4, FP8 = 4, 8
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
DEV = "cuda"


def listed():
    return [
        # Loading a checkpoint: the embedding (= lm_head) matrix of the large shape to 4 bits.
        dict(name="quantise-embedding", op="quantise", rows=49152, cols=2048, type="f16", format=FP4),
        # The attention output of a batched decode step, before the output projection.
        dict(name="quantise-batch64", op="quantise", rows=64, cols=2048, type="f32", format=FP8),
        # One token's attention output, small shape, to 4 bits.
        dict(name="quantise-token", op="quantise", rows=1, cols=576, type="f32", format=FP4),
        # The norm before each linear layer: one token (small shape), a batch of decoding
        # sequences, and a long prompt (large shape).
        dict(name="norm-token", op="norm", rows=1, cols=576, type="f32"),
        dict(name="norm-batch64", op="norm", rows=64, cols=2048, type="f16"),
        dict(name="norm-prompt8192", op="norm", rows=8192, cols=2048, type="f32"),
        # Single-token decode: the logits of the small shape and the down projection of the
        # large one, whose result joins the residual stream.
        dict(name="product-token-lm-head", op="product", n=1, rows=49152, cols=576, x_format=FP8, epilogue="store", type="f32"),
        dict(name="product-token-down", op="product", n=1, rows=2048, cols=8192, x_format=FP8, epilogue="add", type="f32"),
        # A decode step of 64 sequences: q, k and v of the large shape together.
        dict(name="product-batch64-qkv", op="product", n=64, rows=6144, cols=2048, x_format=FP8, epilogue="store", type="f32"),
        # Ragged sizes, as a sharded or pruned layer has them, everything in 4 bits.
        dict(name="product-ragged", op="product", n=37, rows=1003, cols=1100, x_format=FP4, epilogue="store", type="bf16"),
        # Prompts: gate and up of the large shape with SwiGLU, handed on in 8 bits; and the same
        # matrix as a plain product with everything in 4 bits.
        dict(name="product-prompt4096-swiglu", op="product", n=4096, rows=16384, cols=2048, x_format=FP8, epilogue="swiglu", type="mx"),
        dict(name="product-prompt8192-fp4", op="product", n=8192, rows=16384, cols=2048, x_format=FP4, epilogue="store", type="f16"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm; half of them on a round step."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and v >= 64:
        v = v // 32 * 32
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["quantise", "norm", "product", "product"])
    if op != "product":
        while True:
            rows, cols = _spread(rng, 1, 49152), _spread(rng, 32, 16384)
            if rows * cols <= (49152 * 2048 if op == "quantise" else 8192 * 2048):
                break
        c = dict(op=op, rows=rows, cols=cols, type=rng.choice(["f32", "f16", "bf16"]))
        if op == "quantise":
            c["format"] = rng.choice([FP4, FP8])
        return c
    while True:
        n, rows, cols = _spread(rng, 1, 8192), _spread(rng, 32, 49152), _spread(rng, 32, 16384)
        if n * rows * cols <= 8192 * 16384 * 2048 and n * rows <= 8192 * 16384 and rows * cols <= 49152 * 2048:
            break
    epilogue = rng.choice(["store", "add", "swiglu"])
    kind = "mx" if epilogue == "swiglu" else rng.choice(["f32", "f16", "bf16"])
    return dict(op=op, n=n, rows=rows + rows % 2, cols=cols, x_format=rng.choice([FP8, FP4]), epilogue=epilogue, type=kind)


# ---- MX in plain operations ------------------------------------------------------------------


def _padded(cols):
    return (cols + 127) // 128 * 128


def _tiled(e):
    """Scale bytes [rows][padded / 32] -> tiles, zeros in the rows that fill the last tile."""
    rows, blocks = e.shape
    t = (rows + 127) // 128
    full = torch.zeros(t * 128, blocks, dtype=e.dtype, device=e.device)
    full[:rows] = e
    return full.view(t, 4, 32, blocks // 4, 4).permute(0, 3, 2, 1, 4).reshape(-1)


def _untiled(tiles, rows, cols):
    t, kt = (rows + 127) // 128, _padded(cols) // 128
    return tiles.view(t, kt, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(t * 128, kt * 4)[:rows]


def _quantise(x, fmt):
    """fp32 [rows][cols] -> codes (uint8, or float8_e4m3fn) and scale tiles (uint8)."""
    rows, cols = x.shape
    full = torch.zeros(rows, _padded(cols), dtype=torch.float32, device=x.device)
    full[:, :cols] = x
    blocks = full.view(rows, -1, 32)
    amax = blocks.abs().amax(2)
    # The exponent of the block's largest magnitude, less that of the format's largest value.
    e = (amax.view(torch.int32) >> 23) - 127 - (2 if fmt == FP4 else 8)
    e = e.clamp(-127, 127)
    q = blocks * ((127 - e) << 23).view(torch.float32)[:, :, None]
    tiles = _tiled((e + 127).to(torch.uint8))
    if fmt == FP8:
        return q.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(rows, -1), tiles
    a = q.abs()
    # Halfway cases go to the neighbour whose last bit is zero.
    code = (a > 0.25).to(torch.uint8)
    for above, limit in ((True, 0.75), (False, 1.25), (True, 1.75), (False, 2.5), (True, 3.5), (False, 5.0)):
        code += (a >= limit) if above else (a > limit)
    code += (q < 0).to(torch.uint8) * 8
    code = code.view(rows, -1, 2)
    return code[:, :, 0] | (code[:, :, 1] << 4), tiles


def _values(codes, tiles, rows, cols, fmt, dtype=torch.float32):
    """The values that an MX matrix stands for, [rows][cols]."""
    if fmt == FP8:
        v = codes.to(dtype)
    else:
        grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=dtype, device=codes.device)
        v = grid[torch.stack((codes & 15, codes >> 4), 2).long()].view(rows, -1)
    e = _untiled(tiles, rows, cols).to(torch.int32)
    s = torch.where(e > 0, e << 23, 1 << 22).view(torch.float32).to(dtype)
    return (v.view(rows, -1, 32) * s[:, :, None]).view(rows, -1)[:, :cols]


def _mx(codes, tiles):
    """An 8-bit MX matrix as the values that its two parts stand for."""
    return {"codes": codes.view(torch.float8_e4m3fn), "scales": tiles.view(torch.float8_e8m0fnu)}


# ---- inputs ----------------------------------------------------------------------------------


def _activations(g, rows, cols, dtype):
    """A residual stream: normal, with a few columns that are far larger than the others."""
    x = torch.randn(rows, cols, generator=g, device=DEV)
    big = torch.rand(cols, generator=g, device=DEV) < 0.01
    return torch.where(big, x * 20, x).to(dtype)


def _buffer(n, dtype=torch.uint8):
    return torch.zeros(n, dtype=dtype, device=DEV)


def _mx_buffer(rows, cols, fmt):
    """Room for an MX matrix, zeroed once: codes, scales."""
    return _buffer(rows * _padded(cols) * fmt // 8).view(rows, -1), _buffer((rows + 127) // 128 * (_padded(cols) // 128) * 512)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    c, s = case, {"case": case}
    if c["op"] == "quantise":
        x = _activations(g, c["rows"], c["cols"], torch.float32) if c["format"] == FP8 else 0.02 * torch.randn(c["rows"], c["cols"], generator=g, device=DEV)
        s["x"] = x.to(TYPES[c["type"]])
        s["codes"], s["scales"] = _mx_buffer(c["rows"], c["cols"], c["format"])
        if c["format"] == FP4:
            s["values"] = torch.zeros_like(s["x"])
    elif c["op"] == "norm":
        dtype = TYPES[c["type"]]
        s["x"] = torch.randn(c["rows"], c["cols"], generator=g, device=DEV).to(dtype)
        s["residual"] = _activations(g, c["rows"], c["cols"], dtype)
        s["gain"] = (1 + 0.1 * torch.randn(c["cols"], generator=g, device=DEV)).half()
        s["sum"] = torch.zeros_like(s["x"])
        s["codes"], s["scales"] = _mx_buffer(c["rows"], c["cols"], FP8)
    else:
        n, rows, cols = c["n"], c["rows"], c["cols"]
        s["w"] = _quantise(0.02 * torch.randn(rows, cols, generator=g, device=DEV), FP4)
        s["xq"] = _quantise(_activations(g, n, cols, torch.float32), c["x_format"])
        if c["epilogue"] == "swiglu":
            s["codes"], s["scales"] = _mx_buffer(n, rows // 2, FP8)
        else:
            s["y"] = _buffer(n * rows, TYPES[c["type"]]).view(n, rows)
        if c["epilogue"] == "add":
            s["residual"] = torch.randn(n, rows, generator=g, device=DEV).to(TYPES[c["type"]])
    return s


# ---- one pass --------------------------------------------------------------------------------


def run(s):
    return _own_run(s) if own else _plain_run(s)


def _plain_run(s):
    c = s["case"]
    if c["op"] == "quantise":
        codes, tiles = _quantise(s["x"].float(), c["format"])
        if c["format"] == FP8:
            return _mx(codes, tiles)
        return {"values": _values(codes, tiles, c["rows"], c["cols"], FP4).to(TYPES[c["type"]])}
    if c["op"] == "norm":
        t = s["x"].float() + s["residual"].float()
        y = t * torch.rsqrt((t * t).mean(1, keepdim=True) + 1e-5) * s["gain"].float()
        return {"sum": t.to(TYPES[c["type"]]), **_mx(*_quantise(y, FP8))}
    n, rows, cols = c["n"], c["rows"], c["cols"]
    y = _values(*s["xq"], n, cols, c["x_format"]) @ _values(*s["w"], rows, cols, FP4).t()
    if c["epilogue"] == "swiglu":
        gate, up = y[:, : rows // 2], y[:, rows // 2 :]
        return _mx(*_quantise(gate / (1 + torch.exp(-gate)) * up, FP8))
    if c["epilogue"] == "add":
        y = y + s["residual"].float()
    return {"y": y.to(TYPES[c["type"]])}


_ctx = None


def _framework():
    """The framework's kernel layer and this process's context, made once."""
    global _ctx
    import os
    import sys

    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "opure-voxelengine_b200")
    if _ctx is None:
        if package not in sys.path:
            sys.path.insert(0, package)
        from voxelengine import cuda

        _ctx = cuda, cuda.Ctx(0)
    return _ctx


def _own_run(s):
    cu, ctx = _framework()
    c = s["case"]
    if c["op"] == "quantise":
        q = cu.MxMatrix(s["codes"].data_ptr(), s["scales"].data_ptr(), c["rows"], c["cols"], c["format"])
        t = cu.VALUE_TYPES[c["type"]]
        ctx.mx_quantize(s["x"].data_ptr(), t, c["cols"], q)
        if c["format"] == FP8:
            return _mx(s["codes"], s["scales"])
        ctx.mx_dequantize(q, s["values"].data_ptr(), t, c["cols"])
        return {"values": s["values"]}
    if c["op"] == "norm":
        q = cu.MxMatrix(s["codes"].data_ptr(), s["scales"].data_ptr(), c["rows"], c["cols"], FP8)
        ctx.mx_rmsnorm(cu.MxNormArgs(
            x=s["x"].data_ptr(), x_type=cu.VALUE_TYPES[c["type"]], x_stride=c["cols"], residual=s["residual"].data_ptr(),
            sum=s["sum"].data_ptr(), gain=s["gain"].data_ptr(), eps=1e-5, out=q))
        return {"sum": s["sum"], **_mx(s["codes"], s["scales"])}
    n, rows, cols = c["n"], c["rows"], c["cols"]
    a = cu.MxGemmArgs(
        w=cu.MxMatrix(s["w"][0].data_ptr(), s["w"][1].data_ptr(), rows, cols, FP4),
        x=cu.MxMatrix(s["xq"][0].data_ptr(), s["xq"][1].data_ptr(), n, cols, c["x_format"]))
    if c["epilogue"] == "swiglu":
        a.epilogue = cu.EPI_SWIGLU
        a.out = cu.MxMatrix(s["codes"].data_ptr(), s["scales"].data_ptr(), n, rows // 2, FP8)
        ctx.mx_gemm(a)
        return _mx(s["codes"], s["scales"])
    a.y, a.y_type, a.y_stride = s["y"].data_ptr(), cu.VALUE_TYPES[c["type"]], rows
    if c["epilogue"] == "add":
        a.epilogue, a.residual = cu.EPI_ADD, s["residual"].data_ptr()
    ctx.mx_gemm(a)
    return {"y": s["y"]}


# ---- what a pass cannot do without, and its exact result -----------------------------------------


def _mx_bytes(rows, cols, fmt):
    return rows * cols * fmt / 8 + rows * math.ceil(cols / 32)


def work(case):
    c = case
    if c["op"] == "quantise":
        size = c["rows"] * c["cols"] * SIZE[c["type"]]
        back = _mx_bytes(c["rows"], c["cols"], FP4) + size if c["format"] == FP4 else 0
        return {"bytes": size + _mx_bytes(c["rows"], c["cols"], c["format"]) + back, "flops": 2 * c["rows"] * c["cols"]}
    if c["op"] == "norm":
        size = c["rows"] * c["cols"] * SIZE[c["type"]]
        return {"bytes": 3 * size + 2 * c["cols"] + _mx_bytes(c["rows"], c["cols"], FP8), "flops": 6 * c["rows"] * c["cols"]}
    n, rows, cols = c["n"], c["rows"], c["cols"]
    size = _mx_bytes(n, rows // 2, FP8) if c["epilogue"] == "swiglu" else n * rows * SIZE[c["type"]]
    if c["epilogue"] == "add":
        size *= 2
    return {"bytes": size + _mx_bytes(rows, cols, FP4) + _mx_bytes(n, cols, c["x_format"]), "flops": 2 * n * rows * cols}


def _pow2(e):
    """2^e in float64, for whole e inside its range."""
    return (e.long() + 1023 << 52).view(torch.float64)


def _exact_mx(x, fmt):
    """float64 [rows][cols] -> the values of the codes (padded) and of the scales (tiled), by
    rounding to the step of each value's own binade."""
    low, high, step, top = (0, 2, 1, 6.0) if fmt == FP4 else (-6, 8, 3, 448.0)
    rows, cols = x.shape
    b = torch.nn.functional.pad(x, (0, _padded(cols) - cols)).unflatten(1, (-1, 32))
    m, e = torch.frexp(b.abs().amax(2))
    e = torch.where(m == 0, -127, e - 1 - high).clamp(-127, 127)
    scale = _pow2(e)
    q = b / scale[:, :, None]
    unit = _pow2((torch.frexp(q)[1] - 1).clamp(min=low) - step)
    q = (torch.round(q / unit) * unit).clamp(-top, top)
    t = (rows + 127) // 128
    tiles = torch.full((t * 128, scale.shape[1]), 2.0**-127, dtype=torch.float64, device=x.device)
    tiles[:rows] = scale
    tiles = tiles.unflatten(1, (-1, 4)).unflatten(0, (t, 4, 32)).permute(0, 3, 2, 1, 4)
    return q, scale, tiles.flatten()


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "quantise":
        if c["format"] == FP8:
            q, _, tiles = _exact_mx(s["x"].double(), FP8)
            return {"codes": q.flatten(1), "scales": tiles}
        parts = []
        for part in s["x"].split(8192):
            q, scale, _ = _exact_mx(part.double(), FP4)
            parts.append((q * scale[:, :, None]).flatten(1)[:, : c["cols"]])
        return {"values": torch.cat(parts)}
    if c["op"] == "norm":
        t = s["x"].double() + s["residual"].double()
        y = s["gain"].double() * t / torch.sqrt(t.square().sum(1, keepdim=True) / c["cols"] + 1e-5)
        q, _, tiles = _exact_mx(y, FP8)
        return {"sum": t, "codes": q.flatten(1), "scales": tiles}
    n, rows, cols = c["n"], c["rows"], c["cols"]
    w, x = (_exact_values(*s[k], r, cols, f) for k, r, f in (("w", rows, FP4), ("xq", n, c["x_format"])))
    y = torch.einsum("nk,rk->nr", x, w)
    if c["epilogue"] == "swiglu":
        gate, up = y.tensor_split(2, 1)
        q, _, tiles = _exact_mx(gate * torch.sigmoid(gate) * up, FP8)
        return {"codes": q.flatten(1), "scales": tiles}
    return {"y": y + s["residual"].double() if c["epilogue"] == "add" else y}


def _exact_values(codes, tiles, rows, cols, fmt):
    """The values of an MX matrix in float64, from the fields of its codes."""
    if fmt == FP8:
        b = codes.view(torch.uint8).int()
        sign, field, frac, width, bias = b >> 7, b >> 3 & 15, b & 7, 3, 7
    else:
        b = torch.stack((codes & 15, codes >> 4), 2).flatten(1).int()
        sign, field, frac, width, bias = b >> 3, b >> 1 & 3, b & 1, 1, 1
    v = torch.where(field > 0, frac + (1 << width), frac).double()
    v = v * _pow2(field.clamp(min=1) - bias - width) * (1 - 2 * sign)
    r = torch.arange(rows, device=DEV)[:, None]
    k = torch.arange(_padded(cols) // 32, device=DEV)[None]
    at = (r // 128 * (_padded(cols) // 128) + k // 4) * 512 + r % 32 * 16 + r // 32 % 4 * 4 + k % 4
    scale = _pow2(tiles[at.flatten()].view(rows, -1).int() - 127)
    return (v.unflatten(1, (-1, 32)) * scale[:, :, None]).flatten(1)[:, :cols]
