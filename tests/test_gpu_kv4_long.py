"""Attention over the 4-bit KV cache where a kernel for prompts walks many tiles of 64 keys in one split:
few queries over a long past, and blocks of 256 rows whose halves see different tiles, or one of which
is empty. Against a plain 64-bit implementation, with the bounds of test_gpu_kv4.
"""
import numpy as np
import pytest
import torch

import kv4_reference as ref
from test_gpu_kv4 import TYPES, Dev, attend, bound, ctx, release, tables  # noqa: F401 (fixtures)
from test_gpu_kv4_engine import Forward, prompt
from test_gpu_mx import HALF_ULP, TINY, Rows
from voxelengine import cuda as cu
from voxelengine import engine as ve

pytestmark = pytest.mark.gpu


def random_cache(rng, seqs, pages, n_kv, hd, page, ring=0):
    """Codes of any value, scales from 2^-3 to 1, in every page."""
    table, n_pages = tables(rng, seqs, ring or pages)
    cache = ref.Cache(n_pages, n_kv, hd, page, table, ring)
    cache.pool[:] = rng.integers(0, 256, cache.pool.shape)
    cache.pool[..., 16 * hd :] = rng.integers(0x20, 0x39, cache.pool[..., 16 * hd :].shape)
    return cache


def plain(q, k, v, seen, scale):
    """ref.attention for all queries of a head at once; as it, also the largest score's size and value."""
    m, heads, _ = q.shape
    begin, end = (np.array([s[i] for s in seen])[:, None] for i in (0, 1))
    t = np.arange(k.shape[1])[None]
    there = (t >= begin) & (t < end)
    out, size = np.zeros(q.shape), 0.0
    for h in range(heads):
        kk, vv = k[h // (heads // k.shape[0])], v[h // (heads // k.shape[0])]
        x = np.where(there, q[:, h] @ kk.T * scale, -np.inf)
        w = np.exp(x - x.max(1, keepdims=True))
        out[:, h] = w @ vv / w.sum(1, keepdims=True)
        size = max(size, float((np.abs(q[:, h]) @ np.abs(kk).T).max()) * abs(scale))
    return out, size, float(np.abs(v).max())


def check(ctx, t, group, n_kv, hd, page, past, queries, split=0, ring=0, seed=0, n_q=None, max_ctx=None):
    """Entries of `queries` each after `past` positions; twice, with the same bits."""
    rng = np.random.default_rng(seed)
    heads, total = group * n_kv, [a + b for a, b in zip(past, queries)]
    cache = random_cache(rng, len(past), max((n + page - 1) // page for n in total), n_kv, hd, page, ring)
    dev = Dev(ctx, cache)
    q = Rows(ctx, sum(queries), heads * hd, t)
    x = q.put(rng.standard_normal((sum(queries), heads * hd)) * 1.5).reshape(-1, heads, hd)
    begin = np.concatenate(([0], np.cumsum(queries)))
    outs = [attend(ctx, dev, q, np.arange(len(past)), np.array(past) + 1, begin, n_q or max(queries), heads, hd ** -0.5, max_ctx or max(total), split)
            for _ in range(2)]
    got = outs[0].get().reshape(-1, heads, hd)
    assert np.array_equal(got, outs[1].get().reshape(-1, heads, hd))
    for s, (n, m) in enumerate(zip(past, queries)):
        a, b = begin[s], begin[s + 1]
        k, v = cache.get(s, total[s])
        want, size, top = plain(x[a:b], k, v, [(ref.window_begin(n + j, page, ring), n + j + 1) for j in range(m)], hd ** -0.5)
        single = t != "f32" and (n_q or max(queries)) * group > 16
        d = np.abs(got[a:b] - want)
        assert (d <= bound(t, want, size, top, hd, total[s], single)).all(), (s, float(d.max()))


# Rows (queries x group) of a kv head: 17, 88, 128, 129, 300, 360, 257; keys: tiles of 64 in one split.
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("tiles", [3, 5, 8, 9, 13, 40])
@pytest.mark.parametrize("group,n_kv,queries", [(1, 1, 17), (8, 2, 11), (4, 1, 32), (3, 2, 43), (3, 1, 100), (5, 1, 72), (1, 2, 257)])
def test_few_queries_over_a_long_past(ctx, t, hd, tiles, group, n_kv, queries):
    check(ctx, t, group, n_kv, hd, 64, [max(tiles * 64 - queries - 5, 0)], [queries], split=1 << 20, seed=tiles + queries)


@pytest.mark.parametrize("t,hd", [("f32", 64), ("f32", 128), ("f16", 128), ("bf16", 64)])
@pytest.mark.parametrize("split", [0, 640, 1 << 20])
def test_entries_of_very_different_lengths(ctx, t, hd, split):
    """Long pasts with few queries beside prompts, an entry of one query, and one that starts its sequence."""
    check(ctx, t, 4, 2, hd, 32, [3000, 0, 700, 1500, 40], [20, 261, 1, 64, 33], split=split)


@pytest.mark.parametrize("t,hd", [("f32", 64), ("f32", 128), ("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize("page,ring", [(16, 40), (64, 12), (32, 150)])
def test_windows_that_move_within_a_call(ctx, t, hd, page, ring):
    """The second half of a block of rows begins, and ends, tiles later than the first. (What lies in a page
    of the ring is read as it is now, by both sides.)"""
    check(ctx, t, 1, 2, hd, page, [ring * page + 30, 100], [256, 230], ring=ring, split=1 << 20)


@pytest.mark.parametrize("queries,group,n_q", [(5, 3, 8), (5, 4, 8), (9, 1, 16), (9, 2, 16)])
def test_verify_steps_over_a_long_past(ctx, queries, group, n_q):
    """Drafts of several sequences as the engine passes them: n_q a power of two above what any entry has,
    max_ctx the cache's capacity."""
    check(ctx, "f32", group, 8, 64, 64, [1000, 1700, 2040], [queries, queries, 1], n_q=n_q, max_ctx=4096)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("far", [10.0, 15.0, 17.0])
def test_many_small_probabilities_beside_a_large_one(ctx, t, hd, far):
    """A first key with a score about `far` above all others', whose value is 0: the result is the others' sum, 40,000
    probabilities of exp(-far) or so, each off by 2^-22 of itself (pairs) or 2^-11 (16-bit types) and by 2^-36 of the
    largest, and the scores by the usual."""
    rng = np.random.default_rng(int(far))
    n, m = 40000, 40
    table, n_pages = tables(rng, 1, (n + 127) // 128)
    cache = ref.Cache(n_pages, 1, hd, 128, table)
    for at, scales in ((0, cache.at[2]), (8 * hd, cache.at[3])):
        cache.pool[..., at : at + 8 * hd] = 0x22  # 1.0
        cache.pool[..., scales.ravel()] = 0x38    # 1.0
    k, v = np.zeros((1, hd)), np.zeros((1, hd))
    k[0, 0] = 2.0
    k[0, 1:] = 1.0
    cache.put(0, 0, k, v)
    dev = Dev(ctx, cache)
    q = Rows(ctx, m, hd, t)
    x = np.zeros((m, hd))
    x[:, 0] = far  # exact in every type
    q.put(x)
    got = attend(ctx, dev, q, [0], [n - m + 1], [0, m], m, 1, 1.0, n).get()
    # (The first key is kept as 2.0625: its score lies 1.0625 far above the others'.)
    want = plain(x[:, None], *cache.get(0, n), [(0, n - m + 1 + j) for j in range(m)], 1.0)[0][:, 0]
    # The score's own error, 2 far 2^-22 or so, is in all of the others alike; the sums' of n / 64 steps.
    relative = 4 * far * 2.0 ** -22 + 2.0 ** -20 + 2 * (n / 64 + 64) * 2.0 ** -24 + (2.0 ** -11 if t != "f32" else 0.0)
    assert (np.abs(got - want) <= (HALF_ULP[t] + relative) * want + n * 2.0 ** -36 + TINY[t]).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("size", [2.0 ** -30, 1.0, 2.0 ** 12, 2.0 ** 126])
def test_small_queries_beside_a_large_one(ctx, t, hd, size):
    """Scores that come from columns of 2^-20 of the query's largest, whose own column is 0 in every key: held
    to 2^-39 of the largest and so 2^-18 of themselves, where the bound has 2^-22. Up to fp32's largest."""
    if t == "f16" and size not in (1.0, 2.0 ** 12):
        pytest.skip("not values of fp16")
    rng = np.random.default_rng(hd)
    n, m = 300, 40
    cache = random_cache(rng, 1, 5, 1, hd, 64)
    cache.pool[..., cache.at[0][:, 0]] &= 0xF0  # column 0's codes
    dev = Dev(ctx, cache)
    q = Rows(ctx, m, hd, t)
    x = rng.uniform(1, 2, (m, hd)) * rng.choice([-1, 1], (m, hd)) * size
    x[:, 1:] *= 2.0 ** -20
    x = q.put(x)  # as the type has them
    scale = float(np.float32(0.25 / size * 2.0 ** 20))
    got = attend(ctx, dev, q, [0], [n - m + 1], [0, m], m, 1, scale, n).get()
    want, biggest, top = plain(x[:, None], *cache.get(0, n), [(0, n - m + 1 + j) for j in range(m)], scale)
    assert biggest < 100
    d = np.abs(got[:, None] - want)
    assert (d <= bound(t, want, biggest, top, hd, n, t != "f32") + top * 2 * biggest * 2.0 ** -18).all(), float(d.max())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("m", [4, 15, 40])
def test_queries_of_the_largest_size(ctx, t, hd, m):
    """Queries up to fp32's largest and of its subnormals beside ordinary ones; a query with an infinity or NaN is
    NaN, and no other."""
    rng = np.random.default_rng(m)
    n = 200
    cache = random_cache(rng, 1, 4, 1, hd, 64)
    dev = Dev(ctx, cache)
    size = np.array([2.0 ** 125, 2.0 ** 126, 2.0 ** 127, 2.0 ** -128])
    for s in size:
        q = Rows(ctx, m, hd, t)
        x = rng.uniform(0.9, 0.99, (m, hd)) * rng.choice([-1, 1], (m, hd)) * s * 2
        x[1::4, 3], x[2::4, 5] = np.inf, np.nan
        x = q.put(x)
        scale = float(np.float32(2.0 ** -3 / s)) if s > 1 else 2.0 ** 124
        got = attend(ctx, dev, q, [0], [n - m + 1], [0, m], m, 1, scale, n).get()
        ok = np.isfinite(x).all(1)
        want, biggest, top = plain(np.where(ok[:, None], x, 0)[:, None], *cache.get(0, n), [(0, n - m + 1 + j) for j in range(m)], scale)
        # (2^-128 (1 + ..) has 21 bits: held exactly.)
        assert (np.abs(got[ok] - want[ok, 0]) <= bound(t, want, biggest, top, hd, n, t != "f32" and m > 16)[ok, 0]).all()
        assert np.isnan(got[~ok]).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("k_scale,v_scale", [(2.0 ** -7, 8.0), (2.0 ** 40, 2.0 ** -60), (2.0 ** -60, 2.0 ** 10)])
@pytest.mark.parametrize("queries", [3, 40])
def test_tensor_scales(ctx, t, k_scale, v_scale, queries):
    """Powers of two for all keys and all values, taken out of the call's scale again."""
    rng = np.random.default_rng(queries)
    n, heads, hd = 400, 2, 64
    cache = random_cache(rng, 1, 7, 2, hd, 64)
    k, v = cache.get(0, n)
    cache.k_scale, cache.v_scale = k_scale, v_scale
    dev = Dev(ctx, cache)
    q = Rows(ctx, queries, heads * hd, t)
    x = q.put(rng.standard_normal((queries, heads * hd))).reshape(queries, heads, hd)
    got = attend(ctx, dev, q, [0], [n - queries + 1], [0, queries], queries, heads, 0.125 / k_scale, n, 256).get().reshape(queries, heads, hd)
    want, size, top = plain(x, k, v, [(0, n - queries + 1 + j) for j in range(queries)], 0.125)
    if t == "f16":  # as far as it holds them
        want = np.clip(want * v_scale, -65504, 65504) / v_scale
    tiny = 2.0 ** -25 / v_scale if t == "f16" else 0.0
    assert (np.abs(got / v_scale - want) <= bound(t, want, size, top, hd, n, t != "f32") + tiny).all()


def test_entries_without_a_limit_of_queries(ctx):
    """n_q above what there are rows stands for no limit."""
    check(ctx, "f32", 2, 2, 64, 64, [300, 500], [3, 4], n_q=2 ** 32 - 1)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group,queries", [(3, 3), (4, 4), (16, 1), (17, 1), (1, 17)])
def test_both_sides_of_the_choice_of_kernel(ctx, t, hd, group, queries):
    """Up to 16 rows of a kv head probabilities of 16-bit types are pairs too, above one rounding to fp16."""
    check(ctx, t, group, 2, hd, 32, [700, 90], [queries, 1], seed=group)


@pytest.mark.parametrize("queries", [1, 30])
@pytest.mark.parametrize("max_ctx", [0, 1, 256, 600])
def test_an_understated_max_ctx_is_reported(ctx, queries, max_ctx):
    """More keys than the splits that max_ctx asks for hold: reported; what was written is of the rows alone."""
    rng = np.random.default_rng(1)
    dev = Dev(ctx, random_cache(rng, 1, 20, 2, 64, 64))
    q = Rows(ctx, queries, 2 * 64, "f32")
    q.put(rng.standard_normal((queries, 128)))
    out = attend(ctx, dev, q, [0], [1280 - queries + 1], [0, queries], queries, 2, 0.125, max_ctx)
    assert ctx.last_error() == cu.ERR_DEVICE_BOUNDS
    out.get()


def test_one_scratch_for_calls_of_any_shape(ctx):
    """Zeroed once: each call leaves the counters as the next one needs them, whatever its shape."""
    rng = np.random.default_rng(4)
    n_kv, hd, keys = 2, 64, 1500
    cache = random_cache(rng, 3, 24, n_kv, hd, 64)
    dev = Dev(ctx, cache)
    kv = [cache.get(s, keys) for s in range(3)]
    shapes = [(3, 1, 2, 256), (1, 40, 4, 128), (3, 4, 2, 512), (3, 1, 6, 0), (2, 100, 2, 256), (1, 1, 2, 256), (3, 7, 4, 0), (1100, 1, 4, 256), (3, 1, 2, 256)]
    need = max(cu.kv4_attention_scratch_bytes(n, n * m, m, heads, n_kv, hd, keys, split) for n, m, heads, split in shapes)
    scratch = ctx.buffer(need).fill(0)
    for n, m, heads, split in shapes:
        q = Rows(ctx, n * m, heads * hd, "f32")
        x = q.put(rng.standard_normal((n * m, heads * hd))).reshape(n, m, heads, hd)
        seq = np.arange(n) % 3
        got = attend(ctx, dev, q, seq, np.full(n, keys - m + 1), None, m, heads, 0.125, keys, split, scratch=scratch).get().reshape(n, m, heads, hd)
        for i in list(range(min(n, 3))) + [n - 1]:
            want, size, top = plain(x[i], *kv[seq[i]], [(0, keys - m + 1 + j) for j in range(m)], 0.125)
            assert (np.abs(got[i] - want) <= bound("f32", want, size, top, hd, keys)).all(), (n, m, heads, split, i)


# ---- through the engine -----------------------------------------------------------------------------

WIDE = dict(vocab=1000, hidden=2048, inter=512, layers=2, heads=32, kv_heads=8, max_pos=4096)


@pytest.fixture(scope="module")
def wide(tmp_path_factory):
    path = ve.synth_model(str(tmp_path_factory.mktemp("kv4long") / "m"), seed=21, **WIDE)
    return path, Forward(path, WIDE)


@pytest.mark.parametrize("chunk,n", [(1024, 600), (512, 600), (512, 1037)])
def test_scores_of_long_prompts(wide, chunk, n):
    """A prompt in one chunk whose last block of rows is part-filled, and short last chunks after long ones.
    Log probabilities differ by at most twice what logits do."""
    path, fwd = wide
    p = prompt(7, WIDE, n)
    y, tol = fwd.bounded(p)
    with ve.Engine(path, max_len=4096, kv=ve.KV_FP4, prefill_chunk=chunk) as eng:
        got = eng.score([p])[0]["logprobs"]
        tokens, _ = eng.generate([p], 3)
    lp = y - y.max(1, keepdims=True)
    lp -= np.log(np.exp(lp).sum(1, keepdims=True))
    assert np.abs(got[1:] - lp[np.arange(n - 1), p[1:]]).max() <= 2 * tol
    assert len(tokens[0]) == 3 and fwd.follows(p, tokens[0])


def test_speculation_after_long_prompts(wide):
    path, fwd = wide
    prompts = [prompt(30 + i, WIDE, 1000) for i in range(3)]
    with ve.Engine(path, max_batch=18, max_len=4096, kv=ve.KV_FP4, prefill_chunk=512) as t:
        with ve.Engine(path, max_batch=18, max_len=4096, share=t, kv=ve.KV_FP4) as d:
            got, _, _ = t.spec_generate(d, prompts, 12, k=5)
    for p, g in zip(prompts, got):
        assert len(g) == 12 and fwd.follows(p, g)


def test_scores_of_many_lengths_share_their_scratch(wide):
    """Chunks of 40 different lengths: the splits' sums of each take some 10 MB, in buffers that all share.
    What is left to grow is the step graphs, below 2 MB each."""
    path, _ = wide
    p = prompt(9, WIDE, 300)
    with ve.Engine(path, max_len=4096, kv=ve.KV_FP4, prefill_chunk=256) as eng:
        first = eng.score([p])[0]["logprobs"]
        eng.score([p[:258]])
        free = torch.cuda.mem_get_info(0)[0]
        for n in range(100, 260, 4):
            got = eng.score([p[:n]])[0]["logprobs"]
            assert np.abs(got - first[:n]).max() <= 2e-2
        assert free - torch.cuda.mem_get_info(0)[0] < 40 * (2 << 20) + (40 << 20)
        assert np.array_equal(eng.score([p])[0]["logprobs"], first)


def test_scores_of_a_window(wide):
    """Sequences that fit the window score as without one; longer ones are refused."""
    path, _ = wide
    p = prompt(10, WIDE, 200)
    with ve.Engine(path, max_len=1024, kv=ve.KV_FP4, prefill_chunk=64, page_size=32, kv_window=256) as eng:
        got = eng.score([p], 3)[0]
        with pytest.raises(cu.OpureError):
            eng.score([prompt(11, WIDE, 400)])
        again = eng.score([p], 3)[0]
    with ve.Engine(path, max_len=1024, kv=ve.KV_FP4, prefill_chunk=64, page_size=32) as eng:
        want = eng.score([p], 3)[0]
    assert all(np.array_equal(got[k], again[k]) for k in got)
    assert np.abs(got["logprobs"] - want["logprobs"]).max() <= 2e-2
