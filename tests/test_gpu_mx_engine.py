"""The engine over 4-bit microscaled weights against a numpy forward of the same definition.

The forward below keeps every sum in 64 bits and quantises where the engine does: weights per
block of 32 input columns (4 bits), the input of every linear layer (8 bits). The engine's fp32
sums can move a value across a rounding boundary of its 8-bit code, so logits are compared with
the engine tests' bound (2e-2), and tokens where the forward's two best logits are further apart
than twice that.
"""
import numpy as np
import pytest

import mx_reference as mx
import oracle
from voxelengine import cuda as cu
from voxelengine import engine as ve

pytestmark = pytest.mark.gpu
TOL = 2e-2
# Feed-forward and projection sizes that end inside tiles and blocks' groups; grouped KV heads.
SPEC = dict(vocab=1000, hidden=192, inter=336, layers=2, heads=3, kv_heads=1, max_pos=512)


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    return ve.synth_model(str(tmp_path_factory.mktemp("mx") / "m"), seed=11, **SPEC)


class Forward:
    def __init__(self, path):
        t = {k: v[2].view(np.float16).astype(np.float64) for k, v in oracle.read_safetensors(path + "/model.safetensors").items()}
        self.embed, self.final = t["model.embed_tokens.weight"], t["model.norm.weight"]
        self.layers = []
        for i in range(SPEC["layers"]):
            p = f"model.layers.{i}."
            w = [t[p + f"self_attn.{n}_proj.weight"] for n in "qkvo"] + [t[p + f"mlp.{n}_proj.weight"] for n in ("gate", "up", "down")]
            w = [mx.values(*mx.quantize(m, mx.FP4), m.shape[1], mx.FP4) for m in w]
            self.layers.append((t[p + "input_layernorm.weight"], t[p + "post_attention_layernorm.weight"], w))

    @staticmethod
    def act(x):
        return mx.values(*mx.quantize(x, mx.FP8), x.shape[1], mx.FP8)

    @staticmethod
    def norm(x, g):
        return x / np.sqrt((x * x).mean(1, keepdims=True) + 1e-5) * g

    @staticmethod
    def rope(v, heads):
        n, hd = v.shape[0], v.shape[1] // heads
        v = v.reshape(n, heads, hd // 2, 2)
        a = np.arange(n)[:, None] * 10000.0 ** (-2.0 * np.arange(hd // 2) / hd)
        c, s = np.cos(a)[:, None], np.sin(a)[:, None]
        return np.stack([v[..., 0] * c - v[..., 1] * s, v[..., 0] * s + v[..., 1] * c], 3).reshape(n, heads, hd)

    def logits(self, tokens):
        """Of every position, [n][vocab]."""
        H, G = SPEC["heads"], SPEC["kv_heads"]
        x = self.embed[np.asarray(tokens)]
        n = len(tokens)
        future = np.triu(np.ones((n, n), bool), 1)
        for g1, g2, (wq, wk, wv, wo, wg, wu, wd) in self.layers:
            a = self.act(self.norm(x, g1))
            q = self.rope(a @ wq.T, H)
            k = self.rope(a @ wk.T, G).astype(np.float16).astype(np.float64)
            v = (a @ wv.T).reshape(n, G, -1).astype(np.float16).astype(np.float64)
            out = np.empty_like(q)
            for h in range(H):
                s = np.where(future, -np.inf, q[:, h] @ k[:, h * G // H].T)
                p = np.exp(s - s.max(1, keepdims=True))
                out[:, h] = p / p.sum(1, keepdims=True) @ v[:, h * G // H]
            x = x + self.act(out.reshape(n, -1)) @ wo.T
            a = self.act(self.norm(x, g2))
            g, u = a @ wg.T, a @ wu.T
            x = x + self.act(g / (1 + np.exp(-g)) * u) @ wd.T
        return self.norm(x, self.final) @ self.embed.T

    def follows(self, prompt, got):
        """Whether `got` is a greedy continuation, up to the first choice that is too close."""
        all_tokens = list(prompt) + [int(t) for t in got]
        y = self.logits(all_tokens)
        for i, t in enumerate(got):
            row = y[len(prompt) + i - 1]
            best = int(row.argmax())
            if int(t) != best:
                return row[best] - row[int(t)] < 2 * TOL
        return True


@pytest.fixture(scope="module")
def forward(model):
    return Forward(model)


def test_logits_and_poison(model, forward):
    prompt = [int(t) for t in ve.prompt(1, SPEC["vocab"], 9)]
    with ve.Engine(model, max_len=64, weights=ve.WEIGHTS_MXFP4) as eng:
        assert eng.info.weights == ve.WEIGHTS_MXFP4
        got = eng.forward_logits(prompt)
        want = forward.logits(prompt)[-1]
        assert np.abs(got - want).max() <= TOL
        eng.poison(float("nan"))
        assert np.array_equal(eng.forward_logits(prompt), got)
        with ve.Engine(model, max_len=64) as plain:
            assert plain.info.weights == ve.WEIGHTS_STORED
            assert eng.info.stream_bytes < plain.info.stream_bytes and eng.info.weight_bytes < plain.info.weight_bytes
            # 4-bit weights are another model: closer to their own forward than to the stored one's.
            assert np.abs(got - want).max() < np.abs(plain.forward_logits(prompt) - want).max()


@pytest.mark.parametrize("n_seq,prompt_len,chunk", [(1, 5, 0), (2, 7, 0), (5, 6, 0), (20, 12, 0), (2, 150, 256), (3, 40, 64)])
def test_tokens(model, forward, n_seq, prompt_len, chunk):
    """One token at a time, batches of every product kernel's range, and chunked prefill."""
    prompts = [[int(t) for t in ve.prompt(20 + i, SPEC["vocab"], prompt_len)] for i in range(n_seq)]
    with ve.Engine(model, max_batch=n_seq, max_len=256, weights=ve.WEIGHTS_MXFP4, prefill_chunk=chunk) as eng:
        out, _ = eng.generate(prompts, 5)
    for p, got in zip(prompts, out):
        assert forward.follows(p, got)


def test_refusals(model, tmp_path):
    with pytest.raises(cu.OpureError):
        ve.Engine(model, weights=ve.WEIGHTS_MXFP4, path=ve.PATH_FUSED)
    with pytest.raises(cu.OpureError):
        ve.Engine(model, weights=7)
    int8 = ve.synth_model(str(tmp_path / "q"), seed=3, int8=True, **SPEC)
    with pytest.raises(cu.OpureError):
        ve.Engine(int8, weights=ve.WEIGHTS_MXFP4)
