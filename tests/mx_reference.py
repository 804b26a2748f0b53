"""Microscaled matrices in numpy and 64 bits, from the format's definition: the tests' oracle."""
from __future__ import annotations

import numpy as np

FP4, FP8 = 4, 8


def _positive(exp_bits, man_bits, codes):
    """The values of the codes 0 .. codes - 1 (sign bit clear)."""
    c = np.arange(codes)
    e, m = c >> man_bits, c & ((1 << man_bits) - 1)
    bias = (1 << (exp_bits - 1)) - 1
    return np.where(e > 0, (m + (1 << man_bits)) * 2.0 ** (e - bias - man_bits), m * 2.0 ** (1 - bias - man_bits))


# E2M1: 0 .. 6; E4M3: 0 .. 448 (code 127 is NaN).
GRID = {FP4: _positive(2, 1, 8), FP8: _positive(4, 3, 127)}
EMAX = {FP4: 2, FP8: 8}


def kp(cols):
    return -(-cols // 128) * 128


def scale_offsets(rows, cols):
    """Byte offset of the scale of (row, block), [rows][kp / 32]."""
    r, b = np.arange(rows)[:, None], np.arange(kp(cols) // 32)[None]
    return ((r // 128) * (kp(cols) // 128) + b // 4) * 512 + r % 32 * 16 + r // 32 % 4 * 4 + b % 4


def round_to_grid(a, fmt):
    """Codes of the magnitudes a (64 bits): nearest, ties to the even code, limited."""
    g = GRID[fmt]
    mid = (g[1:] + g[:-1]) / 2
    lo, hi = np.searchsorted(mid, a, "left"), np.searchsorted(mid, a, "right")
    return np.where(lo == hi, lo, np.where(lo % 2 == 0, lo, hi))


def quantize(x, fmt):
    """x [rows][cols] (64 bits) -> (codes [rows][row bytes], scale bytes [rows][kp / 32])."""
    rows, cols = x.shape
    b = np.zeros((rows, kp(cols)))
    b[:, :cols] = x
    b = b.reshape(rows, -1, 32)
    bad = ~np.isfinite(b).all(2)
    b = np.where(bad[:, :, None], 0.0, b)
    m = np.abs(b).max(2)
    byte = np.maximum(np.frexp(m)[1] - 1 - EMAX[fmt], -127) + 127
    byte = np.where(m == 0, 0, byte)
    q = b / 2.0 ** (byte[:, :, None] - 127.0)
    code = round_to_grid(np.abs(q), fmt) + np.where(np.signbit(q), 8 if fmt == FP4 else 128, 0)
    code = np.where(bad[:, :, None], 0, code).reshape(rows, -1).astype(np.uint8)
    byte = np.where(bad, 255, byte).astype(np.uint8)
    if fmt == FP4:
        code = code[:, ::2] | (code[:, 1::2] << 4)
    return code, byte


def values(code, byte, cols, fmt):
    """What codes and scale bytes stand for, [rows][cols] in 64 bits."""
    if fmt == FP4:
        code = np.stack([code & 15, code >> 4], 2).reshape(code.shape[0], -1)
        table = np.concatenate([GRID[FP4], -GRID[FP4]])
    else:
        table = np.concatenate([GRID[FP8], [np.nan], -GRID[FP8], [np.nan]])
    s = np.where(byte == 255, np.nan, 2.0 ** (byte.astype(np.float64) - 127))
    v = table[code].reshape(code.shape[0], -1, 32) * s[:, :, None]
    return v.reshape(code.shape[0], -1)[:, :cols]


def tiles(byte, cols, fill=0):
    """Scale bytes [rows][kp / 32] in the tiled layout; `fill` in the rows that fill a tile."""
    rows = byte.shape[0]
    out = np.full(-(-rows // 128) * (kp(cols) // 128) * 512, fill, np.uint8)
    out[scale_offsets(rows, cols)] = byte
    return out


def untile(t, rows, cols):
    return t[scale_offsets(rows, cols)]
