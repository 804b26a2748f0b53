"""4-bit KV cache and token scores: the calls that are measured, and their plain forms.

A cache in 4 bits keeps a row (the key or value of one position and kv head) as E2M1 codes, two in a
byte, and one E4M3 scale for each 16 of its columns: the scale is the block's largest magnitude
divided by 6, rounded to E4M3 (at most 448), and the codes are the values divided by the rounded
scale, rounded to the nearest code, ties to even, at most 6 in magnitude. A page of one kv head is
page_size / 16 groups of 16 positions, 18 * head_dim bytes each:

  keys' codes    [head_dim / 64][8 g][4 c][2 u] x 8 bytes: position 8 u + g, columns 16 c .. 16 c + 15
  values' codes  [head_dim / 64][8 g][4 c][4 t] x 4 bytes: position 2 c + t % 2 + 8 (t / 2), columns 8 g .. 8 g + 7
  keys' scales   [head_dim / 64][8 g][4 c][2 u]: position 8 u + g, block c
  values' scales [head_dim / 64][4 b][4 c][4 t]: position 2 c + t % 2 + 8 (t / 2), block b

(columns within a panel of 64; the even column of a byte in its low half). A pool is [page][kv head]
of such pages, and a table gives each sequence's pages.

Three operators, over the head layouts of the two model shapes that this framework serves (9 heads
over 3 kv heads, and 32 over 32, head_dim 64) and generic ones:

  append     rotates the queries and keys of token vectors to their positions and appends keys and
             values to the cache in 4 bits; the rotated queries come back, and the cache's values at
             those positions (one more call, the inverse operator).
  attention  softmax(scale q K^T) V over such a cache: single tokens, a few tokens of each sequence
             (verifying drafts), and prompts, causal within a sequence.
  score      from logits: log probabilities and ranks of given tokens, the entropy, and the most
             likely alternatives with their log probabilities.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
DEV = "cuda"
THETA = 10000.0
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # One decoded token of the small shape.
        dict(name="append-token", op="append", seqs=1, each=1, past=4000, heads=9, kv=3, hd=64, page=64, type="f32"),
        # A decode step of 64 sequences, large shape.
        dict(name="append-batch64", op="append", seqs=64, each=1, past=4096, heads=32, kv=32, hd=64, page=64, type="f32"),
        # Two prompts of the large shape.
        dict(name="append-prompt", op="append", seqs=2, each=4096, past=0, heads=32, kv=32, hd=64, page=64, type="f16"),
        # Decode, small shape: one sequence; 64 long ones.
        dict(name="attention-token", op="attention", seqs=1, new=1, past=4000, spread=0, heads=9, kv=3, hd=64, page=64, type="f32"),
        dict(name="attention-batch64-long", op="attention", seqs=64, new=1, past=32768, spread=0, heads=9, kv=3, hd=64, page=64, type="f32"),
        # Decode of 64 sequences, large shape.
        dict(name="attention-batch64", op="attention", seqs=64, new=1, past=4096, spread=0, heads=32, kv=32, hd=64, page=64, type="f32"),
        # A few sequences of very different lengths, wider heads in groups of 4, short pages.
        dict(name="attention-ragged", op="attention", seqs=7, new=1, past=50001, spread=1, heads=32, kv=8, hd=128, page=16, type="bf16"),
        # Verifying 4 drafted tokens of each of 16 sequences.
        dict(name="attention-verify", op="attention", seqs=16, new=5, past=2000, spread=1, heads=9, kv=3, hd=64, page=64, type="f32"),
        # A prompt of the large shape.
        dict(name="attention-prompt", op="attention", seqs=1, new=4096, past=0, spread=0, heads=32, kv=32, hd=64, page=64, type="f32"),
        # One decoded token with its 20 best alternatives; ragged rows; a prompt that is scored.
        dict(name="score-token", op="score", rows=1, vocab=49152, top=20, type="f32"),
        dict(name="score-ragged", op="score", rows=333, vocab=50001, top=8, type="f16"),
        dict(name="score-prompt", op="score", rows=4096, vocab=49152, top=5, type="f32"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm; half of them on a round step."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and v >= 64:
        v = v // 32 * 32
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "attention", "score"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op == "score":
        while True:
            rows, vocab = _spread(rng, 1, 4096), _spread(rng, 1000, 131072)
            if rows * vocab * SIZE[kind] <= 4096 * 49152 * 4:
                return dict(op=op, rows=rows, vocab=vocab, top=rng.choice([0, 1, 3, 5, 8, 10, 20]), type=kind)
    while True:
        kv, group = rng.choice([1, 2, 3, 4, 5, 8, 16, 32]), rng.choice([1, 2, 3, 4, 5, 6, 7, 8])
        hd = rng.choice([64, 64, 128])
        heads = kv * group
        c = dict(op=op, seqs=_spread(rng, 1, 64), heads=heads, kv=kv, hd=hd, page=rng.choice([16, 32, 64, 128]), type=kind)
        if op == "append":
            c["each"], c["past"] = rng.choice([1, 1, _spread(rng, 1, 4096)]), _spread(rng, 1, 100000)
            if c["seqs"] * c["each"] * (heads + 2 * kv) * hd * SIZE[kind] <= 8192 * 6144 * 2 and c["seqs"] * (c["past"] + c["each"]) * kv * hd <= 64 * 32768 * 192:
                return c
            continue
        c["new"] = rng.choice([1, 1, rng.randint(2, 8), _spread(rng, 9, 4096)])
        c["past"], c["spread"] = _spread(rng, 1, 100000), rng.choice([0, 1])
        keys = c["past"] + c["new"]
        if c["seqs"] * keys * kv * hd <= 64 * 32768 * 192 and c["seqs"] * c["new"] * heads * hd * (c["past"] + c["new"] / 2) <= 4096 * 32 * 64 * 2048:
            return c


# ---- the 4-bit form in plain operations ------------------------------------------------------------


def _grid(device, dtype):
    return torch.tensor(GRID + tuple(-v for v in GRID), dtype=dtype, device=device)


def _e4m3(x):
    """float64 >= 0, to the nearest E4M3 value (ties to even), at most 448."""
    unit = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(x, min=2.0**-20))), min=-6.0) - 3.0)
    return torch.clamp(torch.round(x / unit) * unit, max=448.0)


def _quantise(x):
    """float64 [..., 16 n] -> codes (uint8, [..., 16 n]) and scales (float8_e4m3fn, [..., n])."""
    blocks = x.unflatten(-1, (-1, 16))
    scale = _e4m3(blocks.abs().amax(-1) / 6.0)
    q = blocks / torch.where(scale > 0, scale, 1.0)[..., None]
    q = torch.where(scale[..., None] > 0, q, 0.0)
    a = q.abs()
    # Halfway cases go to the neighbour whose last bit is zero.
    code = (a > 0.25).to(torch.uint8)
    for above, limit in ((True, 0.75), (False, 1.25), (True, 1.75), (False, 2.5), (True, 3.5), (False, 5.0)):
        code += (a >= limit) if above else (a > limit)
    code += ((q < 0) & (code > 0)).to(torch.uint8) * 8
    return code.flatten(-2), scale.float().to(torch.float8_e4m3fn)


def _values(codes, scales, dtype):
    """The values that codes and scales stand for."""
    v = _grid(codes.device, dtype)[codes.long()].unflatten(-1, (-1, 16))
    return (v * scales.to(dtype)[..., None]).flatten(-2)


def _pack(kc, ks, vc, vs):
    """Codes [..., 16, hd] and scales [..., 16, hd / 16] of keys and values -> group bytes [..., 18 hd]."""

    def halves(c):
        c = c.unflatten(-1, (-1, 2))
        return c[..., 0] | c[..., 1] << 4

    lead, n = kc.shape[:-2], kc.dim() - 2
    dims = list(range(n))
    hd = kc.shape[-1]
    p = hd // 64

    def order(t, shape, perm):
        return t.reshape(*lead, *shape).permute(*dims, *(n + i for i in perm)).reshape(*lead, -1)

    kcodes = order(halves(kc), (2, 8, p, 4, 8), (2, 1, 3, 0, 4))      # u g p c byte -> p g c u byte
    vcodes = order(halves(vc), (2, 4, 2, p, 8, 4), (3, 4, 1, 0, 2, 5))  # t/2 c t%2 p g byte -> p g c t byte
    kscale = order(ks.view(torch.uint8), (2, 8, p, 4), (2, 1, 3, 0))
    vscale = order(vs.view(torch.uint8), (2, 4, 2, p, 4), (3, 4, 1, 0, 2))
    return torch.cat((kcodes, vcodes, kscale, vscale), -1)


def _unpack(groups, hd):
    """Group bytes [..., 18 hd] -> codes [..., 16, hd] and scales [..., 16, hd / 16] of keys and values."""
    lead, n = groups.shape[:-1], groups.dim() - 1
    dims = list(range(n))
    p = hd // 64

    def order(t, shape, perm, last):
        return t.reshape(*lead, *shape).permute(*dims, *(n + i for i in perm)).reshape(*lead, 16, last)

    def nibbles(b):
        return torch.stack((b & 15, b >> 4), -1).flatten(-2)

    kb, vb, ks, vs = groups.split((8 * hd, 8 * hd, hd, hd), -1)
    kc = nibbles(order(kb, (p, 8, 4, 2, 8), (3, 1, 0, 2, 4), hd // 2))
    vc = nibbles(order(vb, (p, 8, 4, 2, 2, 4), (3, 2, 4, 0, 1, 5), hd // 2))
    ks = order(ks, (p, 8, 4, 2), (3, 1, 0, 2), hd // 16).contiguous().view(torch.float8_e4m3fn)
    vs = order(vs, (p, 4, 4, 2, 2), (3, 2, 4, 0, 1), hd // 16).contiguous().view(torch.float8_e4m3fn)
    return kc, ks, vc, vs


def _sequence(pool, table, case, seq, length, dtype):
    """Keys and values [kv][length][hd] of a sequence, from its pages."""
    hd, page = case["hd"], case["page"]
    pages = table[seq, : (length + page - 1) // page].long()
    groups = pool[pages].transpose(0, 1).reshape(case["kv"], -1, 18 * hd)[:, : (length + 15) // 16]
    kc, ks, vc, vs = _unpack(groups, hd)
    k, v = _values(kc, ks, dtype), _values(vc, vs, dtype)
    return k.flatten(1, 2)[:, :length], v.flatten(1, 2)[:, :length]


def _rotate(x, pos, hd):
    """Pairs (2 i, 2 i + 1) of each head by pos * theta^(-2 i / hd), in float64; x [n][heads][hd]."""
    i = torch.arange(hd // 2, dtype=torch.float64, device=x.device)
    angle = pos.double()[:, None] * torch.exp(-2.0 * i / hd * math.log(THETA))
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = x[..., 0::2].double(), x[..., 1::2].double()
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


# ---- inputs ----------------------------------------------------------------------------------


def _uneven(case, most):
    """A length for each sequence: the largest, or with `spread` even between it and nothing."""
    part = 1 - torch.arange(case["seqs"], dtype=torch.float64, device=DEV) * 0.6180339887498949 % 1
    return (part * most).round().long() if case.get("spread") else torch.full((case["seqs"],), most, device=DEV)


def _cache(case, lengths, g, fill):
    """A pool with its table, pages in any order; with `fill`, rows of every mapped page."""
    hd, page, kv = case["hd"], case["page"], case["kv"]
    need = [(int(n) + page - 1) // page for n in lengths.tolist()]
    total, most = sum(need), max(max(need), 1)
    order = torch.randperm(total, generator=g, device=DEV).int()
    table = torch.full((len(need), most), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at : at + n]
        at += n
    pool = torch.zeros(total, kv, page // 16 * 18 * hd, dtype=torch.uint8, device=DEV)
    if fill:
        # Rotated keys have a few columns that are far larger than the others; values do not.
        big = torch.where(torch.rand(kv, 1, 1, hd, generator=g, device=DEV) < 0.05, 4.0, 1.0)
        step = max(1, (1 << 24) // (kv * page * hd))
        for a in range(0, total, step):
            b = min(total, a + step)
            k = torch.randn(b - a, kv, page // 16, 16, hd, generator=g, device=DEV) * big
            v = torch.randn(b - a, kv, page // 16, 16, hd, generator=g, device=DEV)
            pool[a:b] = _pack(*_quantise(k.double()), *_quantise(v.double())).flatten(2)
    return pool, table


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    c, s = case, {"case": case}
    dtype = TYPES[c["type"]]
    if c["op"] == "score":
        rows, vocab = c["rows"], c["vocab"]
        x = torch.randn(rows, vocab, generator=g, device=DEV) * 2.5
        # A few likely tokens in each row, as a trained model has them; given tokens are often among them.
        at = torch.randint(0, vocab, (rows, 4), generator=g, device=DEV)
        x.scatter_add_(1, at, torch.rand(rows, 4, generator=g, device=DEV) * 16)
        s["logits"] = x.to(dtype)
        other = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
        s["tokens"] = torch.where(torch.rand(rows, generator=g, device=DEV) < 0.8, at[:, 0], other).int()
        top = max(c["top"], 1)
        s["logprob"], s["entropy"] = (torch.zeros(rows, device=DEV) for _ in range(2))
        s["rank"] = torch.zeros(rows, dtype=torch.int32, device=DEV)
        s["top_tokens"] = torch.zeros(rows, top, dtype=torch.int32, device=DEV)
        s["top_logprobs"] = torch.zeros(rows, top, device=DEV)
        return s
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    past = _uneven(c, c["past"])  # positions that each sequence has before this call
    if c["op"] == "append":
        n = c["seqs"] * c["each"]
        s["pool"], s["table"] = _cache(c, past + c["each"], g, False)
        s["seq"] = torch.arange(c["seqs"], device=DEV).repeat_interleave(c["each"]).int()
        s["pos"] = (past[:, None] + torch.arange(c["each"], device=DEV)).flatten().int()
        big = torch.where(torch.rand((heads + 2 * kv) * hd, generator=g, device=DEV) < 0.05, 4.0, 1.0)
        s["qkv"] = (torch.randn(n, (heads + 2 * kv) * hd, generator=g, device=DEV) * big).to(dtype)
        s["q"] = torch.zeros(n, heads * hd, dtype=dtype, device=DEV)
        s["k"], s["v"] = (torch.zeros(n, kv * hd, dtype=dtype, device=DEV) for _ in range(2))
        return s
    new = _uneven(c, c["new"]).clamp(min=1)
    s["pool"], s["table"] = _cache(c, past + new, g, True)
    s["seq"] = torch.arange(c["seqs"], device=DEV).int()
    s["seq_len"] = (past + 1).int()
    s["begin"] = torch.cat((torch.zeros(1, dtype=torch.long, device=DEV), new.cumsum(0))).int()
    rows = int(s["begin"][-1])
    s["rows"], s["max_keys"] = rows, int((past + new).max())
    s["spans"] = [(int(p), int(a), int(b)) for p, a, b in zip(past.tolist(), s["begin"][:-1].tolist(), s["begin"][1:].tolist())]
    s["q"] = (torch.randn(rows, heads * hd, generator=g, device=DEV) * 1.5).to(dtype)
    s["out"] = torch.zeros_like(s["q"])
    return s


# ---- one pass --------------------------------------------------------------------------------


def run(s):
    return _own_run(s) if own else _plain_run(s)


def _scale(c):
    return 1.0 / math.sqrt(c["hd"])


def _plain_run(s):
    c = s["case"]
    if c["op"] == "score":
        return _plain_score(s["logits"], s["tokens"].long(), c["top"])
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    dtype = TYPES[c["type"]]
    if c["op"] == "append":
        n, page = s["qkv"].shape[0], c["page"]
        q, k, v = s["qkv"].view(n, heads + 2 * kv, hd).split((heads, kv, kv), 1)
        q = _rotate(q, s["pos"], hd).float().to(dtype).flatten(1)
        (kc, ks), (vc, vs) = _quantise(_rotate(k, s["pos"], hd)), _quantise(v.double())
        # One position at a time to its place: a group's bytes of that position, and no others.
        groups = s["pool"].view(s["pool"].shape[0], kv, page // 16, 18 * hd)
        pages = s["table"][s["seq"].long(), s["pos"].long() // page].long()
        sub = s["pos"].long() % page // 16
        mine = torch.cat((_halves(kc), _halves(vc), ks.view(torch.uint8), vs.view(torch.uint8)), -1)
        index = _place(hd)[s["pos"].long() % 16]
        groups[pages[:, None, None], torch.arange(kv, device=DEV)[None, :, None], sub[:, None, None], index[:, None]] = mine
        back = groups[pages[:, None, None], torch.arange(kv, device=DEV)[None, :, None], sub[:, None, None], index[:, None]]
        kb, vb, ks, vs = back.split((hd // 2, hd // 2, hd // 16, hd // 16), -1)
        out = [_values(torch.stack((b & 15, b >> 4), -1).flatten(-2), e.contiguous().view(torch.float8_e4m3fn), torch.float32) for b, e in ((kb, ks), (vb, vs))]
        return {"q": q, "k": out[0].to(dtype).flatten(1), "v": out[1].to(dtype).flatten(1)}
    outs = []
    for i, (past, a, b) in enumerate(s["spans"]):
        k, v = _sequence(s["pool"], s["table"], c, i, past + b - a, torch.float32)
        q = s["q"][a:b].float().view(b - a, kv, heads // kv, hd).permute(1, 2, 0, 3).flatten(1, 2)
        x = q @ k.transpose(1, 2) * _scale(c)
        seen = torch.arange(past + b - a, device=DEV)[None, :] <= past + torch.arange(b - a, device=DEV)[:, None]
        x = torch.where(seen.repeat(heads // kv, 1), x, -math.inf)
        x = torch.exp(x - x.amax(-1, keepdim=True))
        o = x @ v / x.sum(-1, keepdim=True)
        outs.append(o.view(kv, heads // kv, b - a, hd).permute(2, 0, 1, 3).reshape(b - a, -1))
    return {"out": torch.cat(outs).to(dtype)}


def _halves(c):
    c = c.unflatten(-1, (-1, 2))
    return c[..., 0] | c[..., 1] << 4


def _place(hd):
    """Where the bytes of a position lie in its group: [16][hd / 2 + hd / 2 + hd / 16 + hd / 16]."""
    b, n = torch.arange(hd // 2, device=DEV), torch.arange(hd // 16, device=DEV)
    t = torch.arange(16, device=DEV)[:, None]
    panel, byte = b // 32, b % 32
    k = panel * 512 + (t % 8) * 64 + byte // 8 * 16 + t // 8 * 8 + byte % 8
    c, j = t % 8 // 2, t % 2 + 2 * (t // 8)
    v = 8 * hd + panel * 512 + byte // 4 * 64 + c * 16 + j * 4 + byte % 4
    ks = 16 * hd + n // 4 * 64 + (t % 8) * 8 + n % 4 * 2 + t // 8
    vs = 17 * hd + n // 4 * 64 + n % 4 * 16 + c * 4 + j
    return torch.cat((k, v, ks, vs), 1)


def _plain_score(logits, tokens, top):
    parts = []
    for x, t in zip(logits.split(512), tokens.split(512)):
        x = x.float()
        m = x.amax(1, keepdim=True)
        e = torch.exp(x - m)
        z = e.sum(1)
        given = x.gather(1, t[:, None])
        ids = torch.arange(x.shape[1], device=DEV)
        ahead = (x > given) | ((x == given) & (ids < t[:, None]))
        part = {
            "logprob": given[:, 0] - m[:, 0] - torch.log(z),
            "rank": ahead.sum(1).int(),
            "entropy": torch.log(z) - (e * (x - m)).sum(1) / z,
        }
        if top:
            value, index = torch.sort(x, dim=1, descending=True, stable=True)
            part["top_tokens"] = index[:, :top].int()
            part["top_logprobs"] = value[:, :top] - m - torch.log(z)[:, None]
        parts.append(part)
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


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
    t = cu.VALUE_TYPES[c["type"]]
    if c["op"] == "score":
        top = c["top"]
        ctx.token_scores(cu.ScoreArgs(
            logits=s["logits"].data_ptr(), type=t, vocab=c["vocab"], rows=c["rows"], stride=c["vocab"], tokens=s["tokens"].data_ptr(),
            logprob=s["logprob"].data_ptr(), rank=s["rank"].data_ptr(), entropy=s["entropy"].data_ptr(), top=top,
            top_tokens=s["top_tokens"].data_ptr() if top else None, top_logprobs=s["top_logprobs"].data_ptr() if top else None))
        out = {k: s[k] for k in ("logprob", "rank", "entropy")}
        return {**out, "top_tokens": s["top_tokens"], "top_logprobs": s["top_logprobs"]} if top else out
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    layout = cu.Kv4Layout(
        pool=s["pool"].data_ptr(), page_table=s["table"].data_ptr(), n_pages=s["pool"].shape[0], max_pages=s["table"].shape[1],
        page_size=c["page"], n_kv=kv, head_dim=hd)
    if c["op"] == "append":
        n = s["qkv"].shape[0]
        ctx.kv4_append(cu.Kv4AppendArgs(
            qkv=s["qkv"].data_ptr(), type=t, stride=s["qkv"].shape[1], q_out=s["q"].data_ptr(), q_stride=heads * hd, seq=s["seq"].data_ptr(),
            pos=s["pos"].data_ptr(), n=n, n_heads=heads, theta=THETA, kv=layout))
        ctx.kv4_read(cu.Kv4ReadArgs(
            k=s["k"].data_ptr(), v=s["v"].data_ptr(), type=t, stride=kv * hd, seq=s["seq"].data_ptr(), pos=s["pos"].data_ptr(), n=n, kv=layout))
        return {k: s[k] for k in ("q", "k", "v")}
    if "scratch" not in s:  # made once and kept, as a program keeps it; its counters start at zero
        need = cu.kv4_attention_scratch_bytes(c["seqs"], s["rows"], c["new"], heads, kv, hd, s["max_keys"])
        s["scratch"] = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
        # On the context's stream, which does not wait for torch's.
        ctx.call("opure_fill", s["scratch"].data_ptr(), 0, s["scratch"].numel())
    ctx.kv4_attention(cu.Kv4AttnArgs(
        q=s["q"].data_ptr(), out=s["out"].data_ptr(), type=t, q_stride=heads * hd, out_stride=heads * hd, seq=s["seq"].data_ptr(),
        seq_len=s["seq_len"].data_ptr(), q_begin=s["begin"].data_ptr() if c["new"] > 1 else None, n=c["seqs"], n_rows=s["rows"], n_q=c["new"], n_heads=heads,
        scale=_scale(c), max_ctx=s["max_keys"], scratch=s["scratch"].data_ptr(), scratch_bytes=s["scratch"].numel(), kv=layout))
    return {"out": s["out"]}


# ---- what a pass cannot do without, and its exact result -----------------------------------------


def work(case):
    c = case
    if c["op"] == "score":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * SIZE[c["type"]] + c["rows"] * (16 + 8 * c["top"]), "flops": 5 * n}
    heads, kv, hd, size = c["heads"], c["kv"], c["hd"], SIZE[c["type"]]
    row = kv * 2 * (hd // 2 + hd // 16)  # a position's keys and values
    if c["op"] == "append":
        n = c["seqs"] * c["each"]
        # Read q, k and v, write q, write the cache, read it again, write its values.
        return {"bytes": n * ((2 * heads + 4 * kv) * hd * size + 2 * row + 8), "flops": n * (3 * (heads + kv) + 4 * kv) * hd}
    part = [1 - i * 0.6180339887498949 % 1 if c["spread"] else 1.0 for i in range(c["seqs"])]
    spans = [(round(p * c["past"]), max(1, round(p * c["new"]))) for p in part]
    rows, keys = sum(n for _, n in spans), sum(p + n for p, n in spans)
    seen = sum(n * p + n * (n + 1) / 2 for p, n in spans)
    return {"bytes": keys * row + 2 * rows * heads * hd * size, "flops": 4 * heads * hd * seen}


def _near(x, low, step, top):
    """float64 to the nearest value of a small format, by the step of each value's own binade."""
    e = torch.frexp(x)[1] - 1
    unit = torch.ldexp(torch.ones_like(x), e.clamp(min=low) - step)
    return (torch.round(x / unit) * unit).clamp(-top, top)


def _exact_rows(x):
    """float64 [..., 16 n] -> the values that its 4-bit form stands for."""
    b = x.reshape(*x.shape[:-1], -1, 16)
    scale = _near(b.abs().max(-1).values / 6, -6, 3, 448.0)[..., None]
    return torch.where(scale > 0, _near(b / scale, 0, 1, 6.0) * scale, 0.0).reshape(x.shape)


def _exact_cache(s, c, seq, length):
    """Keys and values [kv][length][hd] in float64, byte by byte from where the layout has them."""
    hd, page = c["hd"], c["page"]
    t = torch.arange(length, device=DEV)
    groups = s["pool"].view(s["pool"].shape[0], c["kv"], page // 16, 18 * hd)
    rows = groups[s["table"][seq][t // page].long(), :, t % page // 16]  # [length][kv][18 hd]
    rows = rows.gather(2, _place(hd)[t % 16][:, None].expand(-1, c["kv"], -1))
    out = []
    for code, scale in ((rows[..., : hd // 2], rows[..., hd : hd + hd // 16]), (rows[..., hd // 2 : hd], rows[..., hd + hd // 16 :])):
        bits = torch.stack((code % 16, code // 16), -1).flatten(-2).int()
        mag = torch.where(bits % 8 < 2, bits % 8 * 0.5, (2 + bits % 2) * torch.exp2((bits % 8 // 2 - 2).double()))
        e = scale.int()
        mult = torch.where(e < 8, e * 2.0**-9, (8 + e % 8) * torch.exp2((e // 8 - 10).double()))
        v = torch.where(bits >= 8, -mag.double(), mag.double()).unflatten(-1, (-1, 16)) * mult.double()[..., None]
        out.append(v.flatten(-2).transpose(0, 1))
    return out


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "score":
        parts = []
        for x, t in zip(s["logits"].split(256), s["tokens"].long().split(256)):
            x = x.double()
            lp = torch.log_softmax(x, 1)
            mine = lp[torch.arange(len(t), device=DEV), t]
            # Every token's place in the order (larger logits first, equal ones by their index).
            order = torch.argsort(x, dim=1, descending=True, stable=True)
            part = {"logprob": mine, "rank": (order == t[:, None]).int().argmax(1).int(), "entropy": -(torch.exp(lp) * lp).sum(1)}
            if c["top"]:
                best = order[:, : c["top"]]
                part["top_tokens"], part["top_logprobs"] = best.int(), lp.gather(1, best)
            parts.append(part)
        return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    heads, kv, hd = c["heads"], c["kv"], c["hd"]
    if c["op"] == "append":
        n = s["qkv"].shape[0]
        x = s["qkv"].double().reshape(n, -1, hd // 2, 2)
        freq = torch.pow(torch.tensor(THETA, dtype=torch.float64, device=DEV), torch.arange(hd // 2, dtype=torch.float64, device=DEV) * (-2.0 / hd))
        turn = torch.polar(torch.ones_like(freq), freq * s["pos"].double()[:, None])
        turned = torch.view_as_real(torch.view_as_complex(x[:, : heads + kv].contiguous()) * turn[:, None]).reshape(n, heads + kv, hd)
        v = x[:, heads + kv :].reshape(n, kv, hd)
        return {"q": turned[:, :heads].reshape(n, -1), "k": _exact_rows(turned[:, heads:]).reshape(n, -1), "v": _exact_rows(v).reshape(n, -1)}
    outs = []
    for i, (past, a, b) in enumerate(s["spans"]):
        k, v = _exact_cache(s, c, i, past + b - a)
        q = s["q"][a:b].double().view(b - a, kv, -1, hd)
        o = torch.empty_like(q)
        for h in range(kv):
            for r in range(0, b - a, 256):  # queries that see the same keys, a few at a time
                e = min(b - a, r + 256)
                x = torch.einsum("qgd,kd->qgk", q[r:e, h], k[h, : past + e]) * _scale(c)
                hidden = torch.arange(past + e, device=DEV)[None] > past + torch.arange(r, e, device=DEV)[:, None]
                w = torch.softmax(x.masked_fill(hidden[:, None], -math.inf), -1)
                o[r:e, h] = torch.einsum("qgk,kd->qgd", w, v[h, : past + e])
        outs.append(o.reshape(b - a, -1))
    return {"out": torch.cat(outs)}
