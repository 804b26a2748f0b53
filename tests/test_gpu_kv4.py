"""The 4-bit paged KV cache's kernels against a plain 64-bit implementation (kv4_reference).

What the cache holds is compared byte for byte: scales and codes are those of the definition. Bounds
of the others are stated where they are derived.
"""
import numpy as np
import pytest
import torch

import kv4_reference as ref
from test_gpu_mx import HALF_ULP, TINY, Rows
from voxelengine import cuda as cu

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f16", "bf16"]
THETA = 10000.0


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


class Dev:
    """A host cache's copy on the device."""

    def __init__(self, ctx, cache):
        self.cache = cache
        self.pool = ctx.to_device(cache.pool)
        self.table = ctx.to_device(cache.table)
        self.layout = cu.Kv4Layout(
            pool=self.pool.ptr, page_table=self.table.ptr, n_pages=cache.pool.shape[0], max_pages=cache.table.shape[1],
            page_size=cache.page, n_kv=cache.n_kv, head_dim=cache.hd, ring=cache.ring, k_scale=cache.k_scale, v_scale=cache.v_scale)

    def bytes(self):
        return self.pool.download(np.uint8, self.cache.pool.shape)


def tables(rng, seqs, pages, extra=3):
    """Pages of sequences in any order, some of the pool's left over."""
    order = rng.permutation(seqs * pages + extra)[: seqs * pages]
    return order.reshape(seqs, pages).astype(np.int32), seqs * pages + extra


def turned(rng, n, cols):
    x = rng.standard_normal((n, cols))
    x[:, rng.random(cols) < 0.05] *= 8
    return x


# ---- append and read -----------------------------------------------------------------------------


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,n_kv,hd,page,n,shift,ring,k_scale,v_scale", [
    (9, 3, 64, 64, 1, 0, 0, 1.0, 1.0),
    (9, 3, 64, 16, 37, 1, 0, 1.0, 1.0),
    (4, 4, 128, 32, 200, 0, 0, 2.0 ** -7, 8.0),
    (8, 1, 128, 128, 5, 3, 0, 1.0, 1.0),
    (2, 2, 64, 16, 64, 0, 3, 1.0, 1.0),
    (32, 32, 64, 64, 16, 0, 0, 1.0, 0.5),
    (0, 2, 64, 64, 9, 0, 0, 1.0, 1.0),
])
def test_append(ctx, t, heads, n_kv, hd, page, n, shift, ring, k_scale, v_scale):
    rng = np.random.default_rng(n + heads)
    seqs, pages = 3, ring or 8
    table, n_pages = tables(rng, seqs, pages)
    cache = ref.Cache(n_pages, n_kv, hd, page, table, ring, k_scale, v_scale, fill=0xA5)
    dev = Dev(ctx, cache)
    # Every position once; with a ring positions far past it, each page of the ring at most once.
    room = pages * page
    place = rng.choice(seqs * room, n, replace=False)
    seq, pos = place // room, place % room + (5 * room if ring else 0)
    cols = (heads + 2 * n_kv) * hd
    rows = Rows(ctx, n, cols, t, cols + 24 if shift else cols, shift)
    x = rows.put(turned(rng, n, cols))
    q_out = Rows(ctx, n, max(heads * hd, 1), t, heads * hd + 8 * (shift > 0) + (heads == 0), shift)
    seq_d, pos_d = ctx.to_device(seq.astype(np.int32)), ctx.to_device(pos.astype(np.int32))
    ctx.kv4_append(cu.Kv4AppendArgs(
        qkv=rows.ptr, type=cu.VALUE_TYPES[t], stride=rows.stride, q_out=q_out.ptr if heads else None, q_stride=q_out.stride,
        seq=seq_d.ptr, pos=pos_d.ptr, n=n, n_heads=heads, theta=THETA, kv=dev.layout))
    x = x.reshape(n, heads + 2 * n_kv, hd)
    k = ref.rotate(x[:, heads : heads + n_kv], pos, THETA)
    for i in range(n):
        cache.put(seq[i], pos[i], k[i], x[i, heads + n_kv :])
    assert np.count_nonzero(dev.bytes() != cache.pool) == 0
    if heads:
        want = ref.rotate(x[:, :heads], pos, THETA).reshape(n, -1)
        # One rounding to the type (16-bit ones: of the fp32 result), and the angle's error: a few
        # units of 2^-53 of up to pos radians on values of the pair's size.
        bound = (HALF_ULP[t] + 2 * 2.0 ** -24 * (t != "f32")) * np.abs(want) + TINY[t] + np.abs(x).max() * (pos[:, None] + 1) * 2.0 ** -49
        assert (np.abs(q_out.get() - want) <= bound).all()
    # Reading the rows back gives the values that the cache stands for.
    out_k, out_v = (Rows(ctx, n, n_kv * hd, "f32", n_kv * hd + (1 if shift else 0), shift) for _ in range(2))
    ctx.kv4_read(cu.Kv4ReadArgs(k=out_k.ptr, v=out_v.ptr, type=cu.F32, stride=out_k.stride, seq=seq_d.ptr, pos=pos_d.ptr, n=n, kv=dev.layout))
    want_k = ref.values(*ref.quantize(k, k_scale), k_scale).reshape(n, -1)
    want_v = ref.values(*ref.quantize(x[:, heads + n_kv :], v_scale), v_scale).reshape(n, -1)
    assert np.array_equal(out_k.get(), want_k) and np.array_equal(out_v.get(), want_v)


@pytest.mark.parametrize("t", TYPES)
def test_append_special_values(ctx, t):
    """Ties, blocks of zeros, of subnormals, beyond the scale's range, with infinities and NaN; not rotated."""
    hd, n_kv = 64, 2
    cache = ref.Cache(2, n_kv, hd, 16, [[1, 0]])
    dev = Dev(ctx, cache)
    x = np.zeros((3, 2 * n_kv * hd))
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    for b in range(3):
        x[0, 16 * b : 16 * b + 16] = np.concatenate((ties, -ties)) * 2.0 ** (3 * b - 4)
    x[0, 48:64] = np.concatenate((ties, -ties)) * 1.125
    x[0, 80:96] = np.linspace(-6e4, 6e4, 16)
    x[0, 96:112] = np.linspace(-3000, 2600, 16)
    x[0, 112:128] = 2.0 ** -12
    x[1, 3], x[1, 20], x[1, 40], x[1, 70], x[1, 75] = np.inf, np.nan, -np.inf, 1e-3, 5e-3
    x[2] = np.random.default_rng(0).choice(ties, x.shape[1]) * 2.0 ** np.random.default_rng(1).integers(-14, 11, x.shape[1])
    if t != "f16":
        x[1, 128:144], x[1, 150] = 1e38, 1e-38
    rows = Rows(ctx, 3, x.shape[1], t)
    x = rows.put(x)
    seq, pos = ctx.to_device(np.zeros(3, np.int32)), ctx.to_device(np.array([0, 17, 9], np.int32))
    ctx.kv4_append(cu.Kv4AppendArgs(qkv=rows.ptr, type=cu.VALUE_TYPES[t], stride=rows.stride, seq=seq.ptr, pos=pos.ptr, n=3, n_heads=0, theta=0.0, kv=dev.layout))
    for i, p in enumerate((0, 17, 9)):
        cache.put(0, p, x[i, : n_kv * hd].reshape(n_kv, hd), x[i, n_kv * hd :].reshape(n_kv, hd))
    assert np.count_nonzero(dev.bytes() != cache.pool) == 0


def test_append_tiny_tensor_scale(ctx):
    """Values that leave fp32 when divided by the tensor scale saturate like any others."""
    cache = ref.Cache(1, 1, 64, 16, [[0]], k_scale=2.0 ** -60, v_scale=2.0 ** 60)
    dev = Dev(ctx, cache)
    x = np.random.default_rng(3).standard_normal((1, 128)) * 1e30
    rows = Rows(ctx, 1, 128, "f32")
    x = rows.put(x)
    zero = ctx.to_device(np.zeros(1, np.int32))
    ctx.kv4_append(cu.Kv4AppendArgs(qkv=rows.ptr, type=cu.F32, stride=128, seq=zero.ptr, pos=zero.ptr, n=1, n_heads=0, theta=0.0, kv=dev.layout))
    cache.put(0, 0, x[:, :64], x[:, 64:])
    assert np.count_nonzero(dev.bytes() != cache.pool) == 0


def test_append_far_positions_padding_and_in_place(ctx):
    """Positions of a million (a ring), padding vectors left alone, queries rotated in place."""
    heads, n_kv, hd, n = 4, 2, 64, 6
    rng = np.random.default_rng(5)
    cache = ref.Cache(4, n_kv, hd, 16, [[2, 0], [1, 3]], ring=2, fill=0x5A)
    dev = Dev(ctx, cache)
    seq, pos = np.array([0, -1, 1, 0, -7, 1], np.int32), np.array([1000003, 5, 999999, 1000004, -3, 31], np.int32)
    rows = Rows(ctx, n, (heads + 2 * n_kv) * hd, "f32", (heads + 2 * n_kv) * hd + 4)
    x = rows.put(turned(rng, n, rows.cols)).copy()
    ctx.kv4_append(cu.Kv4AppendArgs(qkv=rows.ptr, type=cu.F32, stride=rows.stride, q_out=rows.ptr, q_stride=rows.stride,
                                    seq=ctx.to_device(seq).ptr, pos=ctx.to_device(pos).ptr, n=n, n_heads=heads, theta=THETA, kv=dev.layout))
    want = x.copy().reshape(n, -1, hd)
    live = seq >= 0
    want[live, :heads] = ref.rotate(want[live, :heads], pos[live], THETA)
    k = ref.rotate(x.reshape(n, -1, hd)[:, heads : heads + n_kv], pos, THETA)
    for i in np.nonzero(live)[0]:
        cache.put(seq[i], pos[i], k[i], x.reshape(n, -1, hd)[i, heads + n_kv :])
    # Positions 31 and 999999 of sequence 1 share a slot of the ring, whose bytes are either's.
    differ = dev.bytes() != cache.pool
    page, grp, slot = cache.where(1, 31)
    assert cache.where(1, 999999) == (page, grp, slot)
    for at in cache.at:
        differ[page, :, grp, at[slot]] = False
    assert np.count_nonzero(differ) == 0
    got = rows.get().reshape(n, -1, hd)
    assert np.array_equal(got[~live], want[~live]) and np.array_equal(got[:, heads:], want[:, heads:])
    assert (np.abs(got - want) <= HALF_ULP["f32"] * np.abs(want) + np.abs(x).max() * 1e6 * 2.0 ** -49).all()


def test_bad_pages_are_reported(ctx):
    cache = ref.Cache(2, 1, 64, 16, [[1, -1, 2, 0]])
    dev = Dev(ctx, cache)
    rows = Rows(ctx, 1, 192, "f32")
    rows.put(np.ones((1, 192)))
    out = Rows(ctx, 1, 64, "f32")
    for pos in (16, 32, 64, -1):
        seq, p = ctx.to_device(np.zeros(1, np.int32)), ctx.to_device(np.array([pos], np.int32))
        ctx.kv4_append(cu.Kv4AppendArgs(qkv=rows.ptr, type=cu.F32, stride=192, seq=seq.ptr, pos=p.ptr, n=1, n_heads=1, theta=THETA, kv=dev.layout))
        assert ctx.last_error() == cu.ERR_DEVICE_BOUNDS
        ctx.kv4_read(cu.Kv4ReadArgs(k=out.ptr, type=cu.F32, stride=64, seq=seq.ptr, pos=p.ptr, n=1, kv=dev.layout))
        assert ctx.last_error() == cu.ERR_DEVICE_BOUNDS
    assert (dev.bytes() == 0).all()
    out.get()  # nothing written
    q, o = Rows(ctx, 1, 64, "f32"), Rows(ctx, 1, 64, "f32")
    q.put(np.ones((1, 64)))
    scratch = ctx.buffer(1 << 20).fill(0)
    seq, n = ctx.to_device(np.zeros(1, np.int32)), ctx.to_device(np.array([60], np.int32))
    ctx.kv4_attention(cu.Kv4AttnArgs(q=q.ptr, out=o.ptr, q_stride=64, out_stride=64, seq=seq.ptr, seq_len=n.ptr, n=1, n_rows=1, n_q=1, n_heads=1,
                                     scale=1.0, max_ctx=64, scratch=scratch.ptr, scratch_bytes=1 << 20, kv=dev.layout))
    assert ctx.last_error() == cu.ERR_DEVICE_BOUNDS


# ---- attention -------------------------------------------------------------------------------------


def fill_cache(cache, rng, lengths):
    """Rows for each sequence's positions (with a ring: the last ones), written as bytes straight away."""
    for s, n in enumerate(lengths):
        first = max(0, (n - 1) // cache.page - cache.ring + 1) * cache.page if cache.ring else 0
        for p in range(first, n):
            k = rng.standard_normal((cache.n_kv, cache.hd))
            k[:, ::13] *= 4
            cache.put(s, p, k, rng.standard_normal((cache.n_kv, cache.hd)))


def attend(ctx, dev, q, seq, seq_len, begin, n_q, heads, scale, max_ctx, split=0, stride=0, graph=False, packed=False, scratch=None):
    """One call; q is Rows. Returns the results' Rows (and the packed operand)."""
    n, rows = len(seq), q.rows
    hd, n_kv = dev.cache.hd, dev.cache.n_kv
    out = Rows(ctx, rows, heads * hd, q.t, heads * hd + stride, q.shift)
    need = cu.kv4_attention_scratch_bytes(n, rows, n_q, heads, n_kv, hd, max_ctx, split)
    s = scratch or ctx.buffer(need).fill(0)
    pk = ctx.buffer(cu.packed_bytes(rows, heads * hd)).fill(0) if packed else None
    a = cu.Kv4AttnArgs(
        q=q.ptr, out=out.ptr, type=cu.VALUE_TYPES[q.t], q_stride=q.stride, out_stride=out.stride, seq=ctx.to_device(np.asarray(seq, np.int32)).ptr,
        seq_len=ctx.to_device(np.asarray(seq_len, np.int32)).ptr, q_begin=None if begin is None else ctx.to_device(np.asarray(begin, np.int32)).ptr,
        n=n, n_rows=rows, n_q=n_q, n_heads=heads, scale=scale, max_ctx=max_ctx, split_tokens=split, scratch=s.ptr, scratch_bytes=need,
        kv=dev.layout, out_packed=pk.ptr if pk else None)
    if graph:
        ctx.sync()
        with cu.Graph(ctx) as g:
            ctx.kv4_attention(a)
        for _ in range(3):
            g.launch()
        ctx.sync()
        g.free()
    else:
        for _ in range(2):  # counters are left as they were found
            ctx.kv4_attention(a)
    return (out, pk) if packed else out


def bound(t, want, size, top, hd, keys, single=False):
    """|error| of a result: the scores' (queries held to 2^-23, the sums of hd products in fp32 against the
    sum of magnitudes `size`) and the exponential's (2^-22) go into the weights and their sum, on values of at
    most `top`; sums in fp32 over a chain of at most keys / 64 + 64 steps; `single`: probabilities rounded to
    fp16; the rounding to the type."""
    weights = 2 * size * (2.0 ** -22 + hd * 2.0 ** -24) + 2.0 ** -20 + 2 * (keys / 64 + 64) * 2.0 ** -24 + (2.0 ** -10 if single else 0.0)
    return HALF_ULP[t] * (1 + 2.0 ** -10) * np.abs(want) + TINY[t] + top * weights


def check(ctx, t, heads, n_kv, hd, page, lens, queries, scale, split=0, ring=0, shift=0, stride=0, use_begin=True, graph=False, seed=0, tail=0):
    """Entries with `lens` keys before their queries' own, `queries` each."""
    rng = np.random.default_rng(seed)
    total = [n + m for n, m in zip(lens, queries)]
    pages = ring or max(1, max((x + page - 1) // page for x in total))
    table, n_pages = tables(rng, len(lens), pages)
    if not ring:
        for s, x in enumerate(total):
            table[s, (x + page - 1) // page :] = -1
    cache = ref.Cache(n_pages, n_kv, hd, page, table, ring, fill=0x7F)  # NaN scales wherever nothing was appended
    fill_cache(cache, rng, total)
    dev = Dev(ctx, cache)
    rows = sum(queries) + tail
    q = Rows(ctx, rows, heads * hd, t, heads * hd + stride, shift)
    x = q.put(rng.standard_normal((rows, heads * hd)) * 1.5)
    begin = np.concatenate(([0], np.cumsum(queries)))
    out = attend(ctx, dev, q, np.arange(len(lens)), np.array(lens) + 1, begin if use_begin else None, max(queries), heads, scale,
                 max(max(total), 1), split, stride, graph)
    # Rows behind the last entry's keep their bytes: Rows.get of the whole would see guards there.
    raw, body = out._all()
    if tail:
        assert (body[rows - tail :].view(np.uint8) == 0xA5).all()
    got = out.get()
    for s, (n, m) in enumerate(zip(lens, queries)):
        a, b = begin[s], begin[s + 1]
        k, v = cache.get(s, total[s]) if not ring else ring_rows(cache, s, total[s])
        seen = [(ref.window_begin(n + j, page, ring), n + j + 1) for j in range(m)]
        want, size, top = ref.attention(x[a:b].reshape(m, heads, hd), k, v, seen, scale)
        d = np.abs(got[a:b].reshape(m, heads, hd) - want)
        single = t != "f32" and max(queries) * (heads // n_kv) > 8
        assert (d <= bound(t, want, size, top, hd, total[s], single)).all(), (s, float(d.max()))


def ring_rows(cache, seq, length):
    """Values of the positions that a ring still holds; zeros before them."""
    k = np.zeros((cache.n_kv, length, cache.hd))
    v = k.copy()
    first = ref.window_begin(length - 1, cache.page, cache.ring)
    kk, vv = cache.get(seq, length)
    k[:, first:], v[:, first:] = kk[:, first:], vv[:, first:]
    return k, v


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,n_kv,hd,page,lens", [
    (1, 1, 64, 16, [0]),
    (9, 3, 64, 64, [0, 1, 15, 16, 63, 64, 65]),
    (4, 4, 64, 16, [200, 3]),
    (32, 8, 128, 32, [129, 500]),
    (8, 1, 128, 128, [700, 127, 128]),
    (5, 1, 64, 64, [331]),
    (12, 2, 128, 16, [77, 0]),
    (20, 2, 64, 32, [90]),
])
def test_attention_one_query(ctx, t, heads, n_kv, hd, page, lens):
    check(ctx, t, heads, n_kv, hd, page, lens, [1] * len(lens), hd ** -0.5, use_begin=False)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,n_kv,hd,page,lens,queries", [
    (9, 3, 64, 64, [0, 40, 126], [5, 1, 3]),
    (4, 4, 64, 16, [33, 0, 64], [8, 0, 2]),
    (8, 2, 128, 32, [100, 7], [4, 9]),
    (3, 1, 64, 128, [5], [40]),
])
def test_attention_several_queries(ctx, t, heads, n_kv, hd, page, lens, queries):
    check(ctx, t, heads, n_kv, hd, page, lens, queries, 0.2, tail=2)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("heads,n_kv,hd,page,lens,queries", [
    (1, 1, 64, 64, [0], [17]),
    (2, 2, 64, 64, [0], [128]),
    (1, 1, 64, 16, [0], [300]),
    (6, 2, 64, 32, [100, 0, 30], [150, 0, 33]),
    (4, 1, 64, 128, [257], [65]),
    (2, 1, 128, 64, [0], [260]),
    (8, 4, 128, 16, [70, 1], [40, 129]),
    (5, 1, 128, 128, [63], [26]),
])
def test_attention_prompt(ctx, t, heads, n_kv, hd, page, lens, queries):
    check(ctx, t, heads, n_kv, hd, page, lens, queries, hd ** -0.5, tail=3)


@pytest.mark.parametrize("heads,n_kv,hd,page,ring,lens,queries,split", [
    (2, 2, 64, 128, 3, [520], [100], 0),
    (3, 1, 64, 64, 5, [120, 0], [200, 130], 0),
    (2, 1, 128, 128, 2, [300], [80], 128),
])
def test_attention_prompt_window(ctx, heads, n_kv, hd, page, ring, lens, queries, split):
    """Queries of one page, or of a sequence that fits the ring: later positions of a call would overwrite
    pages that its earlier queries see."""
    check(ctx, "f32", heads, n_kv, hd, page, lens, queries, 0.125, split=split, ring=ring)


@pytest.mark.parametrize("t,hd,split,scale", [("f32", 64, 128, 0.125), ("f32", 128, 256, -0.1), ("f16", 64, 384, 0.3), ("bf16", 128, 128, 0.0)])
@pytest.mark.parametrize("graph", [False, True])
def test_attention_prompt_splits(ctx, t, hd, split, scale, graph):
    check(ctx, t, 4, 2, hd, 64, [500, 0], [90, 140], scale, split=split, graph=graph)


@pytest.mark.parametrize("t", TYPES)
def test_attention_prompt_strides(ctx, t):
    check(ctx, t, 6, 2, 64, 16, [70, 10], [30, 20], 0.125, shift=1, stride=5)


@pytest.mark.parametrize("heads,n_kv,hd,page,ring,lens,queries,split", [
    (9, 3, 64, 16, 3, [100, 20, 47], [1, 1, 1], 0),
    (4, 2, 128, 64, 2, [300, 64], [5, 5], 128),
    (2, 2, 64, 32, 4, [500], [9], 0),
])
def test_attention_window(ctx, heads, n_kv, hd, page, ring, lens, queries, split):
    check(ctx, "f32", heads, n_kv, hd, page, lens, queries, 0.125, split=split, ring=ring)


@pytest.mark.parametrize("hd,split", [(64, 128), (128, 128), (64, 256), (64, 100000)])
@pytest.mark.parametrize("graph", [False, True])
def test_attention_splits(ctx, hd, split, graph):
    check(ctx, "f32", 6, 2, hd, 64, [900, 127, 128, 0], [1, 1, 1, 1], 0.125, split=split, graph=graph)


@pytest.mark.parametrize("t", TYPES)
def test_attention_strides(ctx, t):
    check(ctx, t, 6, 2, 64, 16, [70, 10], [1, 1], 0.125, shift=1, stride=5, use_begin=False)


@pytest.mark.parametrize("scale", [0.0, -0.3, 30.0])
def test_attention_scales(ctx, scale):
    """Uniform weights, a negative scale, and scores so far apart that one key takes all."""
    check(ctx, "f32", 6, 2, 64, 64, [150, 20], [1, 3], scale)


def test_attention_long(ctx):
    check(ctx, "f32", 2, 1, 64, 64, [20000], [1], 0.125)


def simple(rng, n_kv=1, hd=64, page=16, length=40):
    table = np.array([rng.permutation(4)[: (length + page - 1) // page]], np.int32)  # of 4 pages
    cache = ref.Cache(4, n_kv, hd, page, table)
    fill_cache(cache, rng, [length])
    return cache


def test_attention_padding_and_empty_rows(ctx):
    """Entries without a sequence, with no keys or a negative number of them, give zeros; so do the first
    queries of an entry whose keys only the later ones see."""
    rng = np.random.default_rng(1)
    cache = simple(rng)
    dev = Dev(ctx, cache)
    q = Rows(ctx, 7, 64, "f32")
    x = q.put(rng.standard_normal((7, 64)))
    out = attend(ctx, dev, q, [-1, 0, 0, 0], [5, 0, -2, 9], [0, 1, 2, 6, 7], 4, 1, 0.125, 16).get()
    k, v = cache.get(0, 40)
    assert (out[0:5] == 0).all()  # no sequence; none; queries at -2, -1 and 0
    want, size, top = ref.attention(x[5:7].reshape(2, 1, 64), k, v, [(0, 1), (0, 9)], 0.125)
    assert (np.abs(out[5:7].reshape(2, 1, 64) - want) <= bound("f32", want, size, top, 64, 16)).all()


def test_attention_nan_reaches_only_who_sees_it(ctx):
    """A NaN value or key at a position that later queries see and earlier ones do not."""
    rng = np.random.default_rng(2)
    cache = simple(rng, page=16, length=24)
    for bad in (np.nan, np.inf):
        k, v = rng.standard_normal((1, 64)), rng.standard_normal((1, 64))
        v[0, 20] = bad
        cache.put(0, 21, k, v)
        k2 = k.copy()
        k2[0, 3] = bad
        cache.put(0, 23, k2, np.ones((1, 64)))
        dev = Dev(ctx, cache)
        q = Rows(ctx, 5, 64, "f32")
        x = q.put(rng.standard_normal((5, 64)))
        out = attend(ctx, dev, q, [0], [20], [0, 5], 5, 1, 0.125, 24).get()
        kk, vv = cache.get(0, 24)
        want, size, top = ref.attention(x[:2].reshape(2, 1, 64), kk, vv, [(0, 20), (0, 21)], 0.125)
        assert (np.abs(out[:2].reshape(2, 1, 64) - want) <= bound("f32", want, size, top, 64, 24)).all()
        assert np.isnan(out[2:4, 16:32]).all() and np.isfinite(out[2:4, :16]).all() and np.isfinite(out[2:4, 32:]).all()
        assert np.isnan(out[4]).all()


def test_attention_prompt_nan_reaches_only_who_sees_it(ctx):
    """NaN values and keys in the middle of a prompt, and queries that have no keys at its start."""
    rng = np.random.default_rng(12)
    n = 200
    cache = simple(rng, page=128, length=n)
    k, v = rng.standard_normal((1, 64)), rng.standard_normal((1, 64))
    v[0, 50] = np.nan
    cache.put(0, 150, k, v)
    k2 = k.copy()
    k2[0, 3] = np.nan
    cache.put(0, 180, k2, np.ones((1, 64)))
    dev = Dev(ctx, cache)
    q = Rows(ctx, n + 5, 64, "f32")
    x = q.put(rng.standard_normal((n + 5, 64)))
    out = attend(ctx, dev, q, [0], [-4], [0, n + 5], n + 5, 1, 0.125, n).get()
    kk, vv = cache.get(0, n)
    assert (out[:5] == 0).all()
    want, size, top = ref.attention(x[5:155].reshape(150, 1, 64), kk, vv, [(0, i + 1) for i in range(150)], 0.125)
    assert (np.abs(out[5:155].reshape(150, 1, 64) - want) <= bound("f32", want, size, top, 64, n)).all()
    assert np.isnan(out[155:185, 48:64]).all() and np.isfinite(out[155:185, :48]).all() and np.isnan(out[185:]).all()


def test_attention_prompt_packed_operand(ctx):
    rng = np.random.default_rng(13)
    cache = simple(rng, n_kv=2, length=40)
    dev = Dev(ctx, cache)
    q = Rows(ctx, 38, 4 * 64, "f32")
    q.put(rng.standard_normal((38, 256)))
    for split in (0, 128):
        out, pk = attend(ctx, dev, q, [0], [2], [0, 38], 38, 4, 0.125, 256 if split else 40, split, packed=True)
        half = pk.download(np.float16, (2, 48, 256)).astype(np.float64)
        got = out.get()
        assert (np.abs(half[0, :38] + half[1, :38] / 2048 - got) <= 2.0 ** -21 * np.abs(got) + 2.0 ** -30).all() and (half[:, 38:] == 0).all()


def test_attention_queries_of_any_size(ctx):
    """Queries from 1e-30 to 1e4 and rows of zeros: their power of two is taken out."""
    rng = np.random.default_rng(3)
    cache = simple(rng)
    dev = Dev(ctx, cache)
    size = np.array([1e-30, 1e-3, 0.0, 1.0, 1e4])
    q = Rows(ctx, 5, 64, "f32")
    x = q.put(rng.standard_normal((5, 64)) * size[:, None])
    k, v = cache.get(0, 40)
    for i, s in enumerate(size):
        scale = 0.125 / s if s else 1.0
        one = Rows(ctx, 1, 64, "f32")
        one.put(x[i : i + 1])
        got = attend(ctx, dev, one, [0], [40], None, 1, 1, scale, 40).get()
        want, sz, top = ref.attention(x[i : i + 1].reshape(1, 1, 64), k, v, [(0, 40)], float(np.float32(scale)))
        assert (np.abs(got.reshape(1, 1, 64) - want) <= bound("f32", want, sz, top, 64, 40)).all()


def test_attention_packed_operand(ctx):
    rng = np.random.default_rng(4)
    cache = simple(rng, n_kv=2, length=40)
    dev = Dev(ctx, cache)
    q = Rows(ctx, 3, 4 * 64, "f32")
    q.put(rng.standard_normal((3, 256)))
    out, pk = attend(ctx, dev, q, [0, 0, 0], [40, 3, 17], None, 1, 4, 0.125, 40, packed=True)
    half = pk.download(np.float16, (2, 16, 256)).astype(np.float64)
    got = out.get()
    assert (np.abs(half[0, :3] + half[1, :3] / 2048 - got) <= 2.0 ** -21 * np.abs(got) + 2.0 ** -30).all() and (half[:, 3:] == 0).all()


def test_attention_pool_past_four_gigabytes(ctx):
    """Pages whose bytes lie past 2^32."""
    rng = np.random.default_rng(6)
    n_kv, hd, page = 8, 128, 128
    each = cu.kv4_page_bytes(n_kv, hd, page)
    n_pages = (5 << 30) // each
    small = ref.Cache(2, n_kv, hd, page, [[0, 1]])
    fill_cache(small, rng, [150])
    pool = ctx.buffer(n_pages * each)
    dev = Dev(ctx, small)
    high = [n_pages - 1, n_pages - 2]
    for i, p in enumerate(high):
        pool.upload(small.pool[i], p * each)
    dev.table.upload(np.array([high], np.int32))
    dev.layout.pool, dev.layout.n_pages = pool.ptr, n_pages
    q = Rows(ctx, 1, n_kv * hd, "f32")
    x = q.put(rng.standard_normal((1, n_kv * hd)))
    out = attend(ctx, dev, q, [0], [150], None, 1, n_kv, 0.09, 150).get()
    k, v = small.get(0, 150)
    want, size, top = ref.attention(x.reshape(1, n_kv, hd), k, v, [(0, 150)], float(np.float32(0.09)))
    assert (np.abs(out.reshape(1, n_kv, hd) - want) <= bound("f32", want, size, top, hd, 150)).all()
    # Appended to and read there as well.
    rows, back = Rows(ctx, 1, 2 * n_kv * hd, "f32"), Rows(ctx, 1, n_kv * hd, "f32")
    xx = rows.put(rng.standard_normal((1, 2 * n_kv * hd)))
    seq, pos = ctx.to_device(np.zeros(1, np.int32)), ctx.to_device(np.array([150], np.int32))
    ctx.kv4_append(cu.Kv4AppendArgs(qkv=rows.ptr, type=cu.F32, stride=rows.stride, seq=seq.ptr, pos=pos.ptr, n=1, n_heads=0, theta=0.0, kv=dev.layout))
    ctx.kv4_read(cu.Kv4ReadArgs(v=back.ptr, type=cu.F32, stride=n_kv * hd, seq=seq.ptr, pos=pos.ptr, n=1, kv=dev.layout))
    assert np.array_equal(back.get(), ref.values(*ref.quantize(xx[:, n_kv * hd :])))


def test_attention_contexts_share_a_gpu(ctx):
    """Two contexts (streams) at once, each with its scratch, give what each gives alone."""
    rng = np.random.default_rng(7)
    table, n_pages = tables(rng, 1, 40)
    cache = ref.Cache(n_pages, 2, 64, 64, table)
    cache.pool[:] = rng.integers(0, 0x60, cache.pool.shape)
    with cu.Ctx(0) as other:
        results = []
        for c in (ctx, other):
            dev = Dev(c, cache)
            q = Rows(c, 1, 4 * 64, "f32")
            q.put(np.random.default_rng(8).standard_normal((1, 256)))
            results.append((c, dev, q))
        outs = [attend(c, dev, q, [0], [2500], None, 1, 4, 0.01, 2560, split=256) for c, dev, q in results]
        a, b = (o.get() for o in outs)
        assert np.array_equal(a, b) and np.isfinite(a).all()


def test_run_together_in_a_graph(ctx):
    """Append and attention as a decode step makes them, captured once and replayed: each replay takes the
    next position from device memory."""
    heads, n_kv, hd, page, steps = 6, 2, 64, 16, 20
    rng = np.random.default_rng(9)
    table, n_pages = tables(rng, 2, 4)
    cache = ref.Cache(n_pages, n_kv, hd, page, table, fill=0x7F)
    dev = Dev(ctx, cache)
    cols = (heads + 2 * n_kv) * hd
    rows, q, out = Rows(ctx, 2, cols, "f32"), Rows(ctx, 2, heads * hd, "f32"), Rows(ctx, 2, heads * hd, "f32")
    seq, pos, length = ctx.to_device(np.arange(2, dtype=np.int32)), ctx.buffer(16), ctx.buffer(16)
    need = cu.kv4_attention_scratch_bytes(2, 2, 1, heads, n_kv, hd, 64)
    scratch = ctx.buffer(need).fill(0)
    append = cu.Kv4AppendArgs(qkv=rows.ptr, type=cu.F32, stride=cols, q_out=q.ptr, q_stride=heads * hd, seq=seq.ptr, pos=pos.ptr, n=2, n_heads=heads, theta=THETA, kv=dev.layout)
    attn = cu.Kv4AttnArgs(q=q.ptr, out=out.ptr, type=cu.F32, q_stride=heads * hd, out_stride=heads * hd, seq=seq.ptr, seq_len=length.ptr, n=2, n_rows=2,
                          n_q=1, n_heads=heads, scale=0.125, max_ctx=64, scratch=scratch.ptr, scratch_bytes=need, kv=dev.layout)
    ctx.sync()
    with cu.Graph(ctx) as g:
        ctx.kv4_append(append)
        ctx.kv4_attention(attn)
    for i in range(steps):
        at = np.array([i, i + 30], np.int32)
        if i == 0:  # sequence 1 starts with 30 positions
            for p in range(30):
                cache.put(1, p, rng.standard_normal((n_kv, hd)), rng.standard_normal((n_kv, hd)))
            dev.pool.upload(cache.pool)
        x = rows.put(rng.standard_normal((2, cols))).reshape(2, -1, hd)
        pos.upload(at)
        length.upload(at + 1)
        g.launch()
        k = ref.rotate(x[:, heads : heads + n_kv], at, THETA)
        qq = ref.rotate(x[:, :heads], at, THETA)
        for s in range(2):
            cache.put(s, at[s], k[s], x[s, heads + n_kv :])
        got = out.get().reshape(2, heads, hd)
        for s in range(2):
            kk, vv = cache.get(s, at[s] + 1)
            want, size, top = ref.attention(qq[s : s + 1], kk, vv, [(0, at[s] + 1)], 0.125)
            # The queries were rounded to fp32 on the way: 2^-24 of each score's size more.
            assert (np.abs(got[s] - want[0]) <= bound("f32", want[0], size * 1.5, top, hd, 64)).all()
    g.free()
    assert np.count_nonzero(dev.bytes() != cache.pool) == 0


# ---- refusals --------------------------------------------------------------------------------------


def test_refusals(ctx):
    """What a call is refused for, with a pool and table that are never followed."""
    buf = ctx.buffer(1 << 16).fill(0)
    zero = ctx.to_device(np.zeros(8, np.int32))

    def layout(**k):
        return cu.Kv4Layout(**{**dict(pool=buf.ptr, page_table=zero.ptr, n_pages=4, max_pages=4, page_size=64, n_kv=2, head_dim=64), **k})

    def append(**k):
        return lambda: ctx.kv4_append(cu.Kv4AppendArgs(**{**dict(qkv=buf.ptr, type=cu.F32, stride=512, q_out=buf.ptr, q_stride=256, seq=zero.ptr, pos=zero.ptr,
                                                                 n=1, n_heads=4, theta=THETA, kv=layout()), **k}))

    def read(**k):
        return lambda: ctx.kv4_read(cu.Kv4ReadArgs(**{**dict(k=buf.ptr, v=buf.ptr, type=cu.F32, stride=128, seq=zero.ptr, pos=zero.ptr, n=1, kv=layout()), **k}))

    def attn(**k):
        return lambda: ctx.kv4_attention(cu.Kv4AttnArgs(**{**dict(
            q=buf.ptr, out=buf.ptr + 8192, type=cu.F32, q_stride=256, out_stride=256, seq=zero.ptr, seq_len=zero.ptr, n=2, n_rows=2, n_q=1, n_heads=4,
            scale=1.0, max_ctx=64, scratch=buf.ptr + 16384, scratch_bytes=32768, kv=layout()), **k}))

    for call in (append, read, attn):
        for k in (dict(page_table=None), dict(pool=None), dict(pool=buf.ptr + 4), dict(n_pages=0), dict(max_pages=0), dict(n_kv=0), dict(k_scale=3.0),
                  dict(v_scale=-1.0), dict(ring=5), dict(v_scale=float("nan"))):
            assert status(call(kv=layout(**k))) == cu.ERR_INVALID_ARG, k
        for k in (dict(page_size=48), dict(head_dim=96), dict(head_dim=32), dict(page_size=256), dict(n_kv=65536)):
            assert status(call(kv=layout(**k))) == cu.ERR_UNSUPPORTED, k
        for k in (dict(type=3), dict(seq=None)):
            assert status(call(**k)) == cu.ERR_INVALID_ARG, k
    for k in (dict(qkv=None), dict(qkv=buf.ptr + 2), dict(stride=511), dict(q_stride=255), dict(n_heads=3), dict(theta=-1.0), dict(theta=float("nan")),
              dict(theta=float("inf")), dict(pos=None)):
        assert status(append(**k)) == cu.ERR_INVALID_ARG, k
    for k in (dict(k=None, v=None), dict(stride=127), dict(v=buf.ptr + 2), dict(pos=None)):
        assert status(read(**k)) == cu.ERR_INVALID_ARG, k
    for k in (dict(q=None), dict(out=None), dict(seq_len=None), dict(scratch=None), dict(scratch=buf.ptr + 8), dict(n_heads=3), dict(n_heads=0),
              dict(q_stride=255), dict(out_stride=255), dict(n_rows=3), dict(q=buf.ptr + 2), dict(n=64, n_rows=64, max_ctx=1 << 20, scratch_bytes=16)):
        assert status(attn(**k)) == cu.ERR_INVALID_ARG, k
    assert status(append(n=0, qkv=None)) == status(read(n=0)) == status(attn(n=0)) == status(attn(n_rows=0)) == cu.OK
    assert cu.kv4_attention_scratch_bytes(1, 1, 1, 3, 2, 64, 64) == 0 and cu.kv4_attention_scratch_bytes(1, 1, 1, 4, 2, 96, 64) == 0
    ctx.sync()


def test_wrong_spans_are_reported(ctx):
    """Entries that claim more rows than there are, run backwards, or pass max_ctx."""
    rng = np.random.default_rng(10)
    dev = Dev(ctx, simple(rng, length=40))
    q = Rows(ctx, 4, 64, "f32")
    q.put(rng.standard_normal((4, 64)))
    for begin, n_q, max_ctx in (([0, 3], 2, 64), ([2, 7], 8, 64), ([3, 1], 4, 64), ([-1, 1], 4, 64), ([0, 2], 2, 0)):
        attend(ctx, dev, q, [0], [8 if max_ctx else 39], begin, n_q, 1, 1.0, max_ctx, split=0 if max_ctx else 0)
        if max_ctx:
            assert ctx.last_error() == cu.ERR_DEVICE_BOUNDS, begin


def status(f):
    try:
        f()
    except cu.OpureError as e:
        return e.status
    return cu.OK
