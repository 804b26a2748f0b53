"""The engine over the 4-bit KV cache, and scores of given tokens, against a numpy forward.

The forward keeps every sum in 64 bits and quantises the rotated keys and the values as the cache does.
The engine's sums are fp32 (their error, 2^-22 of the inputs' size or so, is far below the bounds used
here), so that a key or value near a rounding boundary may get the neighbouring code; what such steps do
to the logits is found from the forward itself, by moving every key and value by up to 2^-18 of its
block's largest before it is quantised (`sway`). Bounds are the engine tests' 2e-2 and twice the sway.
"""
import http.client
import json

import numpy as np
import pytest

import kv4_reference as kv4
import oracle
from voxelengine import cuda as cu
from voxelengine import engine as ve

pytestmark = pytest.mark.gpu
SPEC = dict(vocab=1000, hidden=192, inter=336, layers=2, heads=3, kv_heads=1, max_pos=512)
GROUPED = dict(vocab=515, hidden=512, inter=384, layers=2, heads=4, kv_heads=2, max_pos=512)  # head_dim 128


class Forward:
    def __init__(self, path, spec, window=None):
        self.spec, self.window = spec, window  # (page, ring)
        t = {k: v[2].view(np.float16).astype(np.float64) for k, v in oracle.read_safetensors(path + "/model.safetensors").items()}
        self.embed, self.final = t["model.embed_tokens.weight"], t["model.norm.weight"]
        self.layers = []
        for i in range(spec["layers"]):
            p = f"model.layers.{i}."
            w = [t[p + f"self_attn.{n}_proj.weight"] for n in "qkvo"] + [t[p + f"mlp.{n}_proj.weight"] for n in ("gate", "up", "down")]
            self.layers.append((t[p + "input_layernorm.weight"], t[p + "post_attention_layernorm.weight"], w))

    @staticmethod
    def norm(x, g):
        return x / np.sqrt((x * x).mean(1, keepdims=True) + 1e-5) * g

    def cached(self, x, rng):
        if rng is not None:
            block = np.abs(x.reshape(*x.shape[:-1], -1, 16)).max(-1).repeat(16, -1)
            x = x + block * rng.uniform(-1, 1, x.shape) * 2.0 ** -18
        return kv4.values(*kv4.quantize(x))

    def logits(self, tokens, rng=None):
        """Of every position, [n][vocab]."""
        H, G = self.spec["heads"], self.spec["kv_heads"]
        n = len(tokens)
        pos = np.arange(n)
        x = self.embed[np.asarray(tokens)]
        begin = np.array([kv4.window_begin(p, *self.window) for p in pos]) if self.window else np.zeros(n, int)
        hidden = (pos[None] > pos[:, None]) | (pos[None] < begin[:, None])
        for g1, g2, (wq, wk, wv, wo, wg, wu, wd) in self.layers:
            a = self.norm(x, g1)
            q = kv4.rotate((a @ wq.T).reshape(n, H, -1), pos, 10000.0)
            k = self.cached(kv4.rotate((a @ wk.T).reshape(n, G, -1), pos, 10000.0), rng)
            v = self.cached((a @ wv.T).reshape(n, G, -1), rng)
            out = np.empty_like(q)
            for h in range(H):
                s = np.where(hidden, -np.inf, q[:, h] @ k[:, h * G // H].T)
                p = np.exp(s - s.max(1, keepdims=True))
                out[:, h] = p / p.sum(1, keepdims=True) @ v[:, h * G // H]
            x = x + out.reshape(n, -1) @ wo.T
            a = self.norm(x, g2)
            g, u = a @ wg.T, a @ wu.T
            x = x + (g / (1 + np.exp(-g)) * u) @ wd.T
        return self.norm(x, self.final) @ self.embed.T

    def bounded(self, tokens):
        y = self.logits(tokens)
        sway = max(np.abs(self.logits(tokens, np.random.default_rng(s)) - y).max() for s in range(3))
        return y, 2e-2 + 2 * sway

    def follows(self, prompt, got):
        """Whether `got` is a greedy continuation, up to the first choice that is too close."""
        y, tol = self.bounded(list(prompt) + [int(t) for t in got])
        for i, t in enumerate(got):
            row = y[len(prompt) + i - 1]
            best = int(row.argmax())
            if int(t) != best:
                return row[best] - row[int(t)] < 2 * tol
        return True


@pytest.fixture(scope="module", params=[SPEC, GROUPED], ids=["hd64", "hd128"])
def model(request, tmp_path_factory):
    return ve.synth_model(str(tmp_path_factory.mktemp("kv4") / "m"), seed=11, **request.param), request.param


def prompt(seed, spec, n):
    return [int(t) for t in ve.prompt(seed, spec["vocab"], n)]


def test_logits_and_info(model):
    """Few prompts have a key or value within fp32's error of a rounding boundary (40,000 of them, each
    with a chance of 2^-18 or so): the median error is fp32's own, 1e-3 of the logits' spread at most."""
    path, spec = model
    fwd, errors = Forward(path, spec), []
    with ve.Engine(path, max_len=64, kv=ve.KV_FP4) as eng, ve.Engine(path, max_len=64) as plain:
        assert eng.info.kv == ve.KV_FP4 and plain.info.kv == ve.KV_FP16
        assert eng.info.kv_bytes_per_token * 32 == plain.info.kv_bytes_per_token * 9
        for seed in range(7):
            p = prompt(seed, spec, 40)
            want, tol = fwd.bounded(p)
            got, other = eng.forward_logits(p), plain.forward_logits(p)
            assert np.abs(got - want[-1]).max() <= tol
            errors.append(np.sqrt(np.mean((got - want[-1]) ** 2)) / want[-1].std())
            assert np.abs(other - want[-1]).max() > 2e-2  # 4 bits are not 16
        assert np.median(errors) <= 1e-3, errors
        eng.poison(float("nan"))
        assert np.array_equal(eng.forward_logits(p), got)


@pytest.mark.parametrize("n_seq,prompt_len,chunk,graphs", [(1, 5, 0, True), (2, 7, 0, False), (5, 6, 0, True), (20, 12, 0, True),
                                                          (2, 150, 256, True), (3, 40, 64, True), (3, 41, 50, False)])
def test_tokens(model, n_seq, prompt_len, chunk, graphs):
    """One token at a time, batches, and chunked prefill with several prompts in a step; twice over."""
    path, spec = model
    fwd = Forward(path, spec)
    prompts = [prompt(20 + i, spec, prompt_len - i % 3) for i in range(n_seq)]
    with ve.Engine(path, max_batch=n_seq, max_len=256, kv=ve.KV_FP4, prefill_chunk=chunk, page_size=32, use_graphs=graphs) as eng:
        out, _ = eng.generate(prompts, 5)
        again, _ = eng.generate(prompts, 5)
    assert all(np.array_equal(a, b) for a, b in zip(out, again))
    for p, got in zip(prompts, out):
        assert len(got) == 5 and fwd.follows(p, got)


def test_window(model):
    path, spec = model
    fwd = Forward(path, spec, window=(16, 3))
    with ve.Engine(path, max_len=256, kv=ve.KV_FP4, kv_window=48, page_size=16) as eng:
        for seed in range(2):
            p = prompt(60 + seed, spec, 70)
            assert fwd.follows(p, eng.generate([p], 20)[0][0])


@pytest.mark.parametrize("chunk,top,weights", [(0, 0, 0), (64, 5, 0), (256, 32, 0), (40, 1, 1)])
def test_scores(model, chunk, top, weights):
    """Of several sequences, one of a single token; a decode afterwards is not disturbed. Log
    probabilities differ by at most twice what logits do, the entropy of `vocab` tokens by at most
    2 tol (1 + log vocab)."""
    path, spec = model
    fwd = Forward(path, spec)
    seqs = [prompt(70 + i, spec, n) for i, n in enumerate((33, 1, 57, 2))]
    with ve.Engine(path, max_batch=4, max_len=64, kv=ve.KV_FP4, prefill_chunk=chunk, weights=weights) as eng:
        before, _ = eng.generate(seqs[:1], 4)
        got = eng.score(seqs, top)
        after, _ = eng.generate(seqs[:1], 4)
        assert np.array_equal(before[0], after[0])
    for s, o in zip(seqs, got):
        assert o["logprobs"].shape == (len(s),)
        assert o["logprobs"][0] == 0 and o["ranks"][0] == 0 and o["entropies"][0] == 0
        if top:
            assert (o["top_tokens"][0] == -1).all() and np.isneginf(o["top_logprobs"][0]).all()
        if weights:
            continue  # another model: only the form is looked at
        y, tol = fwd.bounded(s)
        for t in range(1, len(s)):
            row = y[t - 1]
            lp = row - row.max() - np.log(np.exp(row - row.max()).sum())
            assert abs(o["logprobs"][t] - lp[s[t]]) <= 2 * tol
            assert abs(o["entropies"][t] + (np.exp(lp) * lp).sum()) <= 2 * tol * (1 + np.log(spec["vocab"]))
            above = int((row > row[s[t]] + 2 * tol).sum()), int((row > row[s[t]] - 2 * tol).sum())
            assert above[0] <= o["ranks"][t] <= above[1]
            if top:
                ids = o["top_tokens"][t]
                assert len(set(ids.tolist())) == top and (np.diff(o["top_logprobs"][t]) <= 0).all()
                assert np.abs(o["top_logprobs"][t] - lp[ids]).max() <= 2 * tol
                assert np.abs(o["top_logprobs"][t] - np.sort(lp)[::-1][:top]).max() <= 2 * tol


@pytest.mark.parametrize("chunk", [0, 64])
def test_scores_of_the_fp16_cache(model, chunk):
    """Scores need no 4-bit cache: those of every prefix's own logits."""
    path, spec = model
    s = prompt(5, spec, 12)
    with ve.Engine(path, max_len=64, prefill_chunk=chunk) as eng:
        got = eng.score([s], 3)[0]
        for t in range(1, len(s)):
            row = eng.forward_logits(s[:t]).astype(np.float64)
            lp = row - row.max() - np.log(np.exp(row - row.max()).sum())
            assert abs(got["logprobs"][t] - lp[s[t]]) <= 4e-2
            assert np.abs(got["top_logprobs"][t] - np.sort(lp)[::-1][:3]).max() <= 4e-2


def test_load_kv(model):
    """A context given as rows of fp16, quantised as they are (not rotated), then one token after it."""
    path, spec = model
    H, G = spec["heads"], spec["kv_heads"]
    hd, length = spec["hidden"] // H, 37
    fwd = Forward(path, spec)
    kv = np.random.default_rng(3).standard_normal((spec["layers"], 2, G, length, hd)).astype(np.float16)
    token = prompt(8, spec, 1)[0]

    def logits(rng=None):
        x = fwd.embed[[token]]
        for i, (g1, g2, (wq, wk, wv, wo, wg, wu, wd)) in enumerate(fwd.layers):
            a = fwd.norm(x, g1)
            q = kv4.rotate((a @ wq.T).reshape(1, H, hd), [length], 10000.0)[0]
            own = kv4.rotate((a @ wk.T).reshape(1, G, hd), [length], 10000.0), (a @ wv.T).reshape(1, G, hd)
            k, v = (np.concatenate([fwd.cached(kv[i, j].astype(np.float64), None), fwd.cached(own[j], rng).transpose(1, 0, 2)], 1) for j in (0, 1))
            out = np.empty((H, hd))
            for h in range(H):
                s = k[h * G // H] @ q[h]
                p = np.exp(s - s.max())
                out[h] = p / p.sum() @ v[h * G // H]
            x = x + out.reshape(1, -1) @ wo.T
            a = fwd.norm(x, g2)
            g, u = a @ wg.T, a @ wu.T
            x = x + (g / (1 + np.exp(-g)) * u) @ wd.T
        return (fwd.norm(x, fwd.final) @ fwd.embed.T)[0]

    y = logits()
    tol = 2e-2 + 2 * max(np.abs(logits(np.random.default_rng(s)) - y).max() for s in range(3))
    with ve.Engine(path, max_len=128, kv=ve.KV_FP4, page_size=16) as eng:
        for _ in range(2):
            eng.load_kv(0, kv.view(np.uint16), length)
            got = int(np.ravel(eng.decode_step([token], [length]))[0])
            assert y.max() - y[got] < 2 * tol


@pytest.mark.parametrize("n,k", [(1, 4), (3, 5)])
def test_speculation(model, tmp_path, n, k):
    """A verify step's tokens are one entry of several queries; greedy speculation gives a greedy continuation."""
    path, spec = model
    fwd = Forward(path, spec)
    draft = ve.synth_model(str(tmp_path / "d"), seed=12, **{**spec, "layers": 1})
    prompts = [prompt(90 + i, spec, 11) for i in range(n)]
    with ve.Engine(path, max_batch=n * (k + 1), max_len=96, kv=ve.KV_FP4) as t:
        want, _ = t.generate(prompts, 24)
        for d_path, cache in ((draft, ve.KV_FP16), (path, ve.KV_FP4)):  # few drafts accepted, and most
            with ve.Engine(d_path, max_batch=n * (k + 1), max_len=96, share=t, kv=cache) as d:
                got, st, _ = t.spec_generate(d, prompts, 24, k=k)
            for p, g, w in zip(prompts, got, want):
                assert len(g) == len(w) and fwd.follows(p, g)


@pytest.mark.parametrize("chunk", [0, 16])
def test_server(model, chunk):
    path, spec = model
    p = prompt(3, spec, 9)
    with ve.Engine(path, max_len=64, kv=ve.KV_FP4, prefill_chunk=chunk) as eng:
        want = [int(t) for t in eng.generate([p], 12)[0][0]]
        scores = eng.score([p], 2)[0]
    with ve.Server(path, devices=[0], max_len=64, kv=ve.KV_FP4, prefill_chunk=chunk) as s:
        def post(route, body):
            c = http.client.HTTPConnection("127.0.0.1", s.port, timeout=60)
            c.request("POST", route, json.dumps(body))
            r = c.getresponse()
            out = r.status, json.loads(r.read())
            c.close()
            return out

        st, j = post("/generate", {"tokens": p, "max_tokens": 12})
        assert st == 200 and j["tokens"] == want
        st, j = post("/score", {"tokens": p, "top": 2})
        assert st == 200 and j["logprobs"][0] is None and j["ranks"][1:] == scores["ranks"][1:].tolist()
        np.testing.assert_allclose(j["logprobs"][1:], scores["logprobs"][1:], rtol=1e-6)
        np.testing.assert_allclose(j["entropies"][1:], scores["entropies"][1:], rtol=1e-6)
        assert [t["tokens"] for t in j["top"][1:]] == scores["top_tokens"][1:].tolist()
        np.testing.assert_allclose(j["total_logprob"], scores["logprobs"][1:].sum(), rtol=1e-5)
        assert post("/score", {"tokens": [spec["vocab"]]})[0] == 400
        assert post("/score", {"tokens": p, "top": 33})[0] == 400
        assert "error" in post("/score", {"tokens": p * 10})[1]          # longer than the engine's max_len
        assert post("/score", {"tokens": p[:1]})[1]["logprobs"] == [None]


def test_refusals(model, tmp_path):
    path, spec = model
    with pytest.raises(cu.OpureError):
        ve.Engine(path, kv=ve.KV_FP4, path=ve.PATH_FUSED)
    with pytest.raises(cu.OpureError):
        ve.Engine(path, kv=7)
    small = ve.synth_model(str(tmp_path / "s"), seed=3, **{**SPEC, "heads": 6})  # head_dim 32
    with pytest.raises(cu.OpureError):
        ve.Engine(small, kv=ve.KV_FP4)
    with ve.Engine(path, max_len=32, max_batch=2, kv=ve.KV_FP4) as eng:
        for seqs, top in (([[1] * 33], 0), ([[1]] * 3, 0), ([[spec["vocab"]]], 0), ([[1, 2]], 33), ([[]], 0), ([], 0)):
            with pytest.raises(cu.OpureError):
                eng.score(seqs, top)
        assert eng.score([[1, 2, 3]])[0]["logprobs"].shape == (3,)
