"""opure_token_scores against a plain 64-bit implementation (kv4_reference.scores)."""
import numpy as np
import pytest

import kv4_reference as ref
from test_gpu_mx import Rows
from voxelengine import cuda as cu

pytestmark = pytest.mark.gpu
TYPES = ["f32", "f16", "bf16"]


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


def call(ctx, x, tokens, top, graph=False, want=("logprob", "rank", "entropy", "lse")):
    """x: Rows. Returns a dict of arrays; guards around each are checked."""
    rows, cols = x.rows, x.cols
    bufs = {k: ctx.buffer(4 * rows + 16).fill(0xA5) for k in want}
    tt, tl = ctx.buffer(4 * rows * max(top, 1) + 16).fill(0xA5), ctx.buffer(4 * rows * max(top, 1) + 16).fill(0xA5)
    a = cu.ScoreArgs(logits=x.ptr, type=cu.VALUE_TYPES[x.t], vocab=cols, rows=rows, stride=x.stride, top=top, top_tokens=tt.ptr, top_logprobs=tl.ptr,
                     tokens=None if tokens is None else ctx.to_device(np.asarray(tokens, np.int32)).ptr, **{k: b.ptr for k, b in bufs.items()})
    if graph:
        ctx.sync()
        with cu.Graph(ctx) as g:
            ctx.token_scores(a)
        g.launch()
        g.launch()
        ctx.sync()
        g.free()
    else:
        ctx.token_scores(a)
    out = {}
    for k, b in bufs.items():
        raw = b.download(np.int32, rows + 4)
        assert (raw[rows:].view(np.uint8) == 0xA5).all()
        out[k] = raw[:rows] if k == "rank" else raw[:rows].view(np.float32)
    for k, b, d in (("ids", tt, np.int32), ("best", tl, np.float32)):
        raw = b.download(np.int32, rows * max(top, 1) + 4)
        assert (raw[rows * top :].view(np.uint8) == 0xA5).all()
        out[k] = raw[: rows * top].view(d).reshape(rows, top)
    return out


def check(got, x, tokens, top, rows=None):
    """A sum of exponentials is off by 2^-22 each and by its additions, a chain of at most cols / 512 + 64 of
    them on a thread and across threads (2^-24 each); its logarithm as much, absolutely. Then the roundings
    of the logit's and the maximum's difference, of lse, and of the result. The entropy is a weighted mean
    of x - max with the same errors, on terms whose mean magnitude is |log z| + entropy."""
    for i in range(x.shape[0]) if rows is None else rows:
        lp, rank, ent, lse, ids, best = ref.scores(x[i], -1 if tokens is None else tokens[i], top)
        rel = 2.0 ** -22 + 2 * (x.shape[1] / 512 + 64) * 2.0 ** -24
        if tokens is not None:
            assert got["rank"][i] == rank
            assert abs(got["logprob"][i] - lp) <= rel + 2.0 ** -23 * (abs(lp) + abs(x[i].max() - x[i][tokens[i]])) + 2.0 ** -24
        lz = lse - x[i].max()
        assert abs(got["entropy"][i] - ent) <= 4 * rel * (1 + abs(lz) + abs(ent) + abs(ent - lz))
        assert abs(got["lse"][i] - lse) <= rel + 2.0 ** -23 * abs(lse) + 2.0 ** -24
        assert list(got["ids"][i]) == list(ids)
        assert (np.abs(got["best"][i] - best) <= rel + 2.0 ** -23 * (np.abs(best) + np.abs(best)) + 2.0 ** -24).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols,top,shift,pad", [
    (1, 1, 1, 0, 0), (1, 7, 5, 1, 0), (3, 33, 32, 0, 1), (1, 49152, 20, 0, 0), (5, 50001, 8, 3, 0), (150, 1000, 1, 0, 24), (320, 259, 3, 5, 2),
    (2, 131072, 32, 0, 0), (40, 4096, 16, 0, 0), (40, 4097, 17, 0, 0), (9, 16, 0, 0, 0),
])
def test_scores(ctx, t, rows, cols, top, shift, pad):
    rng = np.random.default_rng(rows * cols)
    x = Rows(ctx, rows, cols, t, cols + pad, shift)
    held = x.put(rng.standard_normal((rows, cols)) * 3 + 12 * (rng.random((rows, cols)) < 2 / cols))
    tokens = np.where(rng.random(rows) < 0.5, held.argmax(1), rng.integers(0, cols, rows))
    got = call(ctx, x, tokens, top)
    check(got, held, tokens, top)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,cols,top,stride", [(1000, 4099, 32, 4099), (900, 9001, 7, 9004), (2, 300007, 20, 300007), (3, 150000, 32, 150000)])
def test_rows_of_every_kind_one_behind_another(ctx, t, rows, cols, top, stride):
    """Rows whose best tokens are gathered in each way follow one another on a CTA: random ones, equal ones,
    rising and falling, large ones that all lie in the words of one thread (32 and 128 threads' strides of words),
    more equal largest ones than any buffer holds. Sizes of more pieces than a thread's 32 bits too."""
    rng = np.random.default_rng(rows + cols)
    vec = 4 if t == "f32" else 8
    i = np.arange(cols)
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    for r in range(rows):
        kind = r % 7
        if kind == 1:
            x[r] = 0.5
        elif kind == 2:
            x[r] = np.sort(x[r])
        elif kind == 3:
            x[r] = np.sort(x[r])[::-1]
        elif kind == 4:
            x[r][i // vec % 128 == r % 128] += 20
        elif kind == 5:
            x[r][i // vec % 32 == r % 32] += 20
        elif kind == 6:
            x[r][rng.permutation(cols)[:700]] = 9.0
    rows_ = Rows(ctx, rows, cols, t, stride)
    held = rows_.put(x)
    tokens = np.where(rng.random(rows) < 0.5, held.argmax(1), rng.integers(0, cols, rows))
    got = call(ctx, rows_, tokens, top)
    again = call(ctx, rows_, tokens, top)
    assert all(np.array_equal(got[k], again[k]) for k in got)
    check(got, held, tokens, top, list(range(min(rows, 30))) + list(range(max(min(rows, 30), rows - 130), rows)))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("cols,stride", [(3, 3), (5, 5), (6, 7), (7, 9), (8, 9), (9, 9), (14, 15)])
def test_short_rows_with_and_without_whole_words(ctx, t, cols, stride):
    """Rows of some of which no aligned 16 bytes are there, in turn with others that have some: many of each on a CTA."""
    rng = np.random.default_rng(cols)
    rows = 6000
    x = Rows(ctx, rows, cols, t, stride)
    held = x.put(rng.standard_normal((rows, cols)) * 4)
    tokens = rng.integers(0, cols, rows)
    got = call(ctx, x, tokens, 3)
    again = call(ctx, x, tokens, 3)
    assert all(np.array_equal(got[k], again[k]) for k in got)
    check(got, held, tokens, 3)


@pytest.mark.parametrize("size", [1e-3, 200.0, 3e4])
def test_scores_of_any_size(ctx, size):
    rng = np.random.default_rng(1)
    x = Rows(ctx, 4, 3001, "f32")
    held = x.put(rng.standard_normal((4, 3001)) * size)
    tokens = held.argmax(1)
    check(call(ctx, x, tokens, 4), held, tokens, 4)


@pytest.mark.parametrize("t", TYPES)
def test_ties_go_to_the_lowest_index(ctx, t):
    """Rows of one value, of two, of zeros with either sign, ascending and descending ones."""
    cols = 20011
    rng = np.random.default_rng(2)
    x = np.stack([np.full(cols, 1.5), rng.integers(0, 2, cols).astype(float), np.where(rng.random(cols) < 0.5, 0.0, -0.0),
                  np.arange(cols) / 512.0, -np.arange(cols) / 512.0, np.full(cols, -1e4)])
    r = Rows(ctx, 6, cols, t)
    held = r.put(x)
    held = held + 0.0  # -0 is 0
    tokens = np.array([777, 13, 20010, 5, 9, 0])
    check(call(ctx, r, tokens, 20), held, tokens, 20)


@pytest.mark.parametrize("t", TYPES)
def test_masked_logits(ctx, t):
    """-inf is a token of probability 0; the type's lowest value too, unless the row holds nothing else."""
    cols = 5000
    low = {"f32": -3.4028234663852886e38, "f16": -65504.0, "bf16": -3.3895313892515355e38}[t]
    rng = np.random.default_rng(3)
    x = rng.standard_normal((5, cols))
    x[0, 100:] = -np.inf
    x[1, 3:] = low
    x[2] = low
    x[3, :] = -np.inf
    x[3, 4999] = 2.0
    x[4, ::2] = -np.inf
    r = Rows(ctx, 5, cols, t)
    held = r.put(x)
    tokens = np.array([3, 1, 4000, 4999, 1])
    got = call(ctx, r, tokens, 8)
    with np.errstate(invalid="ignore"):
        check(got, held, tokens, 8, [2])
        for i in (0, 1, 3, 4):
            lp, rank, ent, lse, ids, best = ref.scores(held[i], tokens[i], 8)
            assert got["rank"][i] == rank and abs(got["logprob"][i] - lp) < 2e-6 and abs(got["lse"][i] - lse) < 2e-6
            assert abs(got["entropy"][i] - ent) < 1e-5 and list(got["ids"][i]) == list(ids)
            f = np.isfinite(best) & (best > -1e4)
            assert np.allclose(got["best"][i][f], best[f], atol=2e-6) and (got["best"][i][~f] < -1e4).all()
    assert (got["best"][3][1:] == -np.inf).all()


def test_nothing_finite_and_nan(ctx):
    cols = 3000
    x = np.zeros((4, cols))
    x[0] = -np.inf
    x[1, 7] = np.nan
    x[2, 9] = np.inf
    x[3] = np.nan
    r = Rows(ctx, 4, cols, "f32")
    r.put(x)
    got = call(ctx, r, [5, 5, 5, 5], 3)
    assert np.isnan(got["logprob"]).all() and np.isnan(got["entropy"]).all()
    assert got["lse"][0] == -np.inf and np.isnan(got["lse"][[1, 3]]).all() and not np.isfinite(got["lse"][2])
    assert list(got["ids"][0]) == [0, 1, 2] and list(got["ids"][1]) == [0, 1, 2] and list(got["ids"][2]) == [9, 0, 1]
    assert list(got["ids"][3]) == [-1] * 3 and (got["best"][3] == -np.inf).all()
    assert got["rank"][0] == 5 and got["rank"][1] == 5 and got["rank"][2] == 6 and got["rank"][3] == 0


def test_no_tokens_and_wrong_ones(ctx):
    rng = np.random.default_rng(4)
    r = Rows(ctx, 3, 1000, "f32")
    held = r.put(rng.standard_normal((3, 1000)))
    got = call(ctx, r, [-1, 5, -9], 2)
    assert got["logprob"][0] == 0 and got["logprob"][2] == 0 and got["rank"][0] == 0 and got["rank"][2] == 0
    check(got, held, [-1, 5, -9], 2, [1])
    got = call(ctx, r, None, 2, want=("entropy", "lse"))
    for i in range(3):
        assert abs(got["lse"][i] - ref.scores(held[i], -1, 2)[3]) < 1e-5
    got = call(ctx, r, [1, 1000, 2], 1)
    assert np.isnan(got["logprob"][1]) and got["rank"][1] == 0 and np.isfinite(got["logprob"][[0, 2]]).all()
    assert ctx.last_error() == cu.ERR_DEVICE_BOUNDS


@pytest.mark.parametrize("rows", [1, 300])
def test_replayed(ctx, rows):
    rng = np.random.default_rng(5)
    r = Rows(ctx, rows, 9000, "f16")
    held = r.put(rng.standard_normal((rows, 9000)))
    tokens = rng.integers(0, 9000, rows)
    check(call(ctx, r, tokens, 6, graph=True), held, tokens, 6)


def test_rows_past_four_gigabytes(ctx):
    """The last row begins past 2^32 bytes."""
    cols, rows, stride = 1000, 3, 1 << 30
    buf = ctx.buffer(4 * (2 * stride + cols))
    rng = np.random.default_rng(6)
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    for i in range(rows):
        buf.upload(x[i], 4 * i * stride)
    lp = ctx.buffer(16)
    ctx.token_scores(cu.ScoreArgs(logits=buf.ptr, type=cu.F32, vocab=cols, rows=rows, stride=stride, tokens=ctx.to_device(np.array([1, 2, 3], np.int32)).ptr, logprob=lp.ptr))
    got = lp.download(np.float32, 3)
    for i in range(rows):
        assert abs(got[i] - ref.scores(x[i].astype(np.float64), i + 1, 0)[0]) < 1e-5


def test_refusals(ctx):
    b = ctx.buffer(4096).fill(0)

    def status(**k):
        try:
            ctx.token_scores(cu.ScoreArgs(**{**dict(logits=b.ptr, type=cu.F32, vocab=100, rows=1, stride=100, lse=b.ptr), **k}))
        except cu.OpureError as e:
            return e.status
        return cu.OK

    for k in (dict(logits=None), dict(logits=b.ptr + 2), dict(type=7), dict(vocab=0), dict(stride=99), dict(top=33, top_tokens=b.ptr, top_logprobs=b.ptr),
              dict(top=5), dict(top=5, top_tokens=b.ptr), dict(vocab=3, top=4, top_tokens=b.ptr, top_logprobs=b.ptr)):
        assert status(**k) == cu.ERR_INVALID_ARG, k
    assert status(rows=1 << 29, stride=1 << 20) == cu.ERR_UNSUPPORTED
    assert status(rows=0, logits=None) == cu.OK and status() == cu.OK
    ctx.sync()
