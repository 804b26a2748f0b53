"""The 4-bit paged KV cache and token scores in plain 64-bit numpy, from their definitions in
opure_cuda.h."""
import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def e4m3_values():
    """The value of each byte without a sign (0x7f: NaN)."""
    b = np.arange(128)
    v = np.where(b < 8, b * 2.0 ** -9, (8 + b % 8) * 2.0 ** (b // 8 - 10.0))
    v[127] = np.nan
    return v


def nearest(x, grid):
    """Index of the nearest grid value, of two equally near ones the even index."""
    i = np.clip(np.searchsorted(grid, x, side="right") - 1, 0, len(grid) - 2)
    low, high = x - grid[i], grid[i + 1] - x
    return np.where((high < low) | ((high == low) & (i % 2 == 1)), i + 1, i)


def quantize(x, tensor=1.0):
    """float64 [..., 16 n] -> codes [..., 16 n] and scale bytes [..., n]."""
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 16)
    bad = ~np.isfinite(b).all(-1)
    b = np.where(bad[..., None], 0.0, b) / tensor
    byte = nearest(np.minimum(np.abs(b).max(-1) / 6, 448.0), e4m3_values()[:127])
    s = e4m3_values()[byte]
    q = np.where(s[..., None] > 0, b / np.where(s > 0, s, 1.0)[..., None], 0.0)
    code = nearest(np.minimum(np.abs(q), 6.0), GRID) + 8 * (np.signbit(b) & (s[..., None] > 0))
    return np.where(bad[..., None], 0, code).reshape(x.shape).astype(np.uint8), np.where(bad, 127, byte).astype(np.uint8)


def values(code, byte, tensor=1.0):
    v = np.where(code & 8, -1.0, 1.0) * GRID[code & 7]
    s = np.where(byte & 128, -1.0, 1.0) * e4m3_values()[byte & 127]
    return (v.reshape(*byte.shape, 16) * s[..., None]).reshape(code.shape) * tensor


def offsets(hd):
    """Byte offsets within a group: of the byte of columns (2 i, 2 i + 1) and of the scale of block b, for
    each of 16 positions: keys' codes [16][hd / 2], values', keys' scales [16][hd / 16], values'."""
    t, i, b = np.arange(16)[:, None], np.arange(hd // 2)[None], np.arange(hd // 16)[None]
    panel, col = i // 32, i % 32 * 2
    kc = panel * 512 + (t % 8) * 64 + col // 16 * 16 + t // 8 * 8 + col % 16 // 2
    c, slot = t % 8 // 2, t % 2 + 2 * (t // 8)
    vc = 8 * hd + panel * 512 + col // 8 * 64 + c * 16 + slot * 4 + col % 8 // 2
    ks = 16 * hd + b // 4 * 64 + (t % 8) * 8 + b % 4 * 2 + t // 8
    vs = 17 * hd + b // 4 * 64 + b % 4 * 16 + c * 4 + slot
    return kc, vc, ks, vs


def rotate(x, pos, theta):
    """x [n][heads][hd], pairs (2 i, 2 i + 1) by pos theta^(-2 i / hd)."""
    hd = x.shape[-1]
    a = np.asarray(pos, np.float64)[:, None] * float(theta) ** (-2.0 * np.arange(hd // 2) / hd)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    out = np.empty(x.shape)
    out[..., 0::2] = x[..., 0::2] * c - x[..., 1::2] * s
    out[..., 1::2] = x[..., 0::2] * s + x[..., 1::2] * c
    return out


class Cache:
    """A pool's bytes [n_pages][n_kv][page / 16][18 hd] on the host."""

    def __init__(self, n_pages, n_kv, hd, page, table, ring=0, k_scale=1.0, v_scale=1.0, fill=0):
        self.pool = np.full((n_pages, n_kv, page // 16, 18 * hd), fill, np.uint8)
        self.table, self.page, self.ring, self.hd, self.n_kv = np.asarray(table, np.int32), page, ring, hd, n_kv
        self.k_scale, self.v_scale = k_scale, v_scale
        self.at = offsets(hd)

    def where(self, seq, pos):
        lp = pos // self.page
        return self.table[seq, lp % self.ring if self.ring else lp], pos % self.page // 16, pos % 16

    def put(self, seq, pos, k, v):
        """Rows k, v [n_kv][hd] in float64."""
        page, grp, t = self.where(seq, pos)
        for x, codes, scales, tensor in ((k, self.at[0], self.at[2], self.k_scale), (v, self.at[1], self.at[3], self.v_scale)):
            code, byte = quantize(x, tensor)
            self.pool[page, :, grp][:, codes[t]] = code[:, 0::2] | code[:, 1::2] << 4
            self.pool[page, :, grp][:, scales[t]] = byte

    def get(self, seq, length):
        """Values [n_kv][length][hd] of positions 0 .. length - 1 (with a ring: of the pages now there)."""
        out = []
        pos = np.arange(length)
        lp = pos // self.page
        page = self.table[seq][lp % self.ring if self.ring else lp]
        rows = self.pool[page, :, pos % self.page // 16]  # [length][n_kv][18 hd]
        t = pos % 16
        for codes, scales, tensor in ((self.at[0], self.at[2], self.k_scale), (self.at[1], self.at[3], self.v_scale)):
            b = np.take_along_axis(rows, codes[t][:, None], 2)
            code = np.stack((b & 15, b >> 4), -1).reshape(length, self.n_kv, self.hd)
            out.append(values(code, np.take_along_axis(rows, scales[t][:, None], 2), tensor).transpose(1, 0, 2))
        return out


def window_begin(p, page, ring):
    return max(0, p // page - ring + 1) * page if ring and p >= 0 else 0


def attention(q, k, v, seen, scale):
    """q [queries][heads][hd], k and v [n_kv][keys][hd], seen [queries] of (begin, end): results, and for the
    bounds the largest scale sum |q| |k| and |v| over what is seen."""
    out = np.zeros(q.shape)
    group = q.shape[1] // k.shape[0]
    size = top = 0.0
    for j, (a, b) in enumerate(seen):
        if b <= a:
            continue
        for h in range(q.shape[1]):
            kk, vv = k[h // group, a:b], v[h // group, a:b]
            x = kk @ q[j, h] * scale
            w = np.exp(x - x.max())
            out[j, h] = w @ vv / w.sum()
            size = max(size, float((np.abs(kk) @ np.abs(q[j, h])).max()) * abs(scale))
            top = max(top, float(np.abs(vv).max()))
    return out, size, top


def scores(x, token, top):
    """One row: log probability, rank, entropy, log-sum-exp, top tokens and their log probabilities."""
    m = x.max()
    e = np.exp(x - m)
    z = e.sum()
    lp = x - m - np.log(z)
    with np.errstate(invalid="ignore"):
        ent = -(e / z * np.where(e > 0, lp, 0.0)).sum()
    order = np.lexsort((np.arange(len(x)), -x))
    rank = int(np.nonzero(order == token)[0][0]) if token >= 0 else 0
    return lp[token] if token >= 0 else 0.0, rank, ent, m + np.log(z), order[:top], lp[order[:top]]
