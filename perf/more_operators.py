"""Cases of the packed-prompt operators: q/k norm, rotary positions and cache
rows of prompts of different lengths packed into one row dimension, their
attention, and the log probabilities of given tokens (from logits, or straight
from the LM head's operands).

`run` computes an operator in its plain form (elementary torch operations in 32
bits) or, where `own` is true, by the framework's entry points."""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = 64  # rows in a block of the paged cache
EPS = 1e-6


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # the first turn of one chat: latency is all
        dict(name="attn 1 of 130", op="attn", B=1, L=130, ragged=False, Hq=16, Hkv=8, D=128,
             dtype="bf16", causal=True, window=-1),
        # a serving batch of short prompts, as the decode benchmark's (512 tokens), ragged
        dict(name="attn 32 to 512", op="attn", B=32, L=512, ragged=True, Hq=16, Hkv=8, D=128,
             dtype="bf16", causal=True, window=-1),
        # documents of very different lengths, four query heads a kv head
        dict(name="attn 6 to 8191", op="attn", B=6, L=8191, ragged=True, Hq=32, Hkv=8, D=128,
             dtype="f16", causal=True, window=-1),
        # one prompt near the rotary table's end: the most work of the set
        dict(name="attn 1 of 32768", op="attn", B=1, L=32768, ragged=False, Hq=16, Hkv=8, D=128,
             dtype="bf16", causal=True, window=-1),
        # 64-dim heads, three query heads a kv head, a sliding window
        dict(name="attn 13 to 3001 window", op="attn", B=13, L=3001, ragged=True, Hq=12, Hkv=4,
             D=64, dtype="bf16", causal=True, window=1023),
        # q/k norm and positions of one short prompt, rows into its cache
        dict(name="rope 1 of 130", op="rope", B=1, L=130, ragged=False, Hq=16, Hkv=8, D=128,
             dtype="bf16", norm=True, cache="rows"),
        # and of a prefill of a whole serving batch into a paged cache
        dict(name="rope 64 to 1024 paged", op="rope", B=64, L=1024, ragged=True, Hq=32, Hkv=8,
             D=128, dtype="f16", norm=True, cache="paged"),
        # the token just decoded, with five alternatives: latency
        dict(name="logprobs 1 x 151936 top 5", op="logprobs", N=1, V=151936, top=5, dtype="bf16",
             temp=1.0),
        # a scored prompt's rows, with the alternatives an API returns
        dict(name="logprobs 4096 x 151936 top 20", op="logprobs", N=4096, V=151936, top=20,
             dtype="bf16", temp=1.0),
        # 32-bit logits of a small vocabulary of odd size, at a sampling temperature
        dict(name="logprobs 301 x 32003 f32", op="logprobs", N=301, V=32003, top=0, dtype="f32",
             temp=0.7),
        # a few tokens against the whole LM head: reading the weights is all
        dict(name="head 7 x 1024 x 151936", op="head", N=7, E=1024, V=151936, dtype="bf16",
             temp=1.0),
        # a scored batch of prompts
        dict(name="head 4096 x 1024 x 151936", op="head", N=4096, E=1024, V=151936, dtype="bf16",
             temp=1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "rope", "logprobs", "logprobs", "head", "head"])
    dtype = rng.choice(["bf16", "f16"])
    Hq, Hkv = rng.choice([(16, 8), (32, 8), (16, 16), (8, 1), (12, 4), (28, 4)])
    D = rng.choice([64, 128, 128])
    if op == "attn":
        c = dict(op=op, B=_log(rng, 1, 64), L=_log(rng, 1, 32768), ragged=rng.random() < 0.8,
                 Hq=Hq, Hkv=Hkv, D=D, dtype=dtype, causal=rng.random() < 0.85, window=-1)
        if c["causal"] and rng.random() < 0.3:
            c["window"] = _log(rng, 16, 4096)
        # no more products than the largest listed case, and 2^19 rows at most
        most = 32768 ** 2 * 16 * 128 / (1 if c["causal"] else 2)
        c["L"] = max(1, min(c["L"], int((most / (c["B"] * Hq * D)) ** 0.5), 2 ** 19 // c["B"]))
        return c
    if op == "rope":
        B = _log(rng, 1, 64)
        L = min(_log(rng, 1, 8192), 64 * 1024 * 48 * 128 // (B * (Hq + 2 * Hkv) * D))
        return dict(op=op, B=B, L=L, ragged=rng.random() < 0.8, Hq=Hq, Hkv=Hkv, D=D, dtype=dtype,
                    norm=rng.random() < 0.7, cache=rng.choice(["none", "rows", "paged"]))
    V = _log(rng, 1000, 151936)
    if op == "logprobs":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        N = min(_log(rng, 1, 16384), 4096 * 151936 * 2 // (V * (4 if dtype == "f32" else 2)))
        return dict(op=op, N=N, V=V, top=rng.choice([0, 1, 5, 20]), dtype=dtype,
                    temp=rng.choice([1.0, 1.0, 0.6]))
    E = 8 * _log(rng, 16, 256)
    N = min(_log(rng, 1, 16384), 4096 * 151936 * 1024 // (V * E))
    return dict(op=op, N=N, E=E, V=V, dtype=dtype, temp=rng.choice([1.0, 1.0, 0.8]))


def lengths(c):
    """The prompts' lengths: all L, or spread over 40 to 100 % of it."""
    if not c["ragged"]:
        return [c["L"]] * c["B"]
    return [max(1, round(c["L"] * (1 - 0.6 * (b * 0.6180339887 % 1)))) for b in range(c["B"])]


# ------------------------------------------------------------------ inputs
def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _drawn(g, logits):
    """A token a row, from the softmax of its logits (the largest of logit + noise)."""
    u = torch.rand(logits.shape, generator=g, device="cuda").clamp_min(1e-30)
    return (logits.float() - (-u.log()).log()).argmax(-1)


def prepare(case, seed):
    c, g = case, torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=c, op=c["op"])
    dt = TYPES[c["dtype"]]
    if c["op"] in ("attn", "rope"):
        Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
        s["lens"] = lens = lengths(c)
        N = sum(lens)
        cu = torch.tensor([0] + lens).cumsum(0)
        s["cu"] = cu.to(torch.int32).cuda()
        qkv = _randn(g, N, (Hq + 2 * Hkv) * D, dtype=dt)
    if c["op"] == "attn":
        s["q"] = 2 * _randn(g, N, Hq, D, dtype=dt)       # scores that prefer some keys
        s["k"] = _randn(g, N, Hkv, D, dtype=dt)
        s["v"] = qkv[:, (Hq + Hkv) * D:].view(N, Hkv, D)  # as the projection leaves it
    elif c["op"] == "rope":
        s["qkv"] = qkv
        s["qn"] = s["kn"] = None
        if c["norm"]:
            s["qn"] = (1 + 0.1 * _randn(g, D)).to(dt)
            s["kn"] = (1 + 0.1 * _randn(g, D)).to(dt)
        inv = 1e6 ** (-torch.arange(0, D, 2, device="cuda") / D)
        ang = torch.arange(max(lens), device="cuda")[:, None] * inv
        ang = torch.cat([ang, ang], 1)
        s["cos"], s["sin"] = ang.cos().half(), ang.sin().half()
        s["table"] = s["kc"] = s["vc"] = None
        if c["cache"] != "none":
            n = -(-max(lens) // BLOCK)
            shape = (c["B"], Hkv, n * BLOCK, D)
            if c["cache"] == "paged":
                s["table"] = torch.randperm(c["B"] * n, generator=g, device="cuda") \
                    .view(c["B"], n).to(torch.int32)
                shape = (c["B"] * n, Hkv, BLOCK, D)
            s["kc"], s["vc"] = _randn(g, *shape, dtype=dt), _randn(g, *shape, dtype=dt)
    elif c["op"] == "logprobs":
        N, V = c["N"], c["V"]
        # a few likely tokens and a long tail
        s["logits"] = x = _randn(g, N, V, dtype=dt).mul_(2.5)
        s["tokens"] = torch.cat([_drawn(g, x[i:i + 256]) for i in range(0, N, 256)])
    else:
        N, E, V = c["N"], c["E"], c["V"]
        s["x"] = _randn(g, N, E, dtype=dt)
        s["w"] = _randn(g, V, E, dtype=dt).mul_(2.5 / math.sqrt(E))
        s["tokens"] = torch.cat([_drawn(g, s["x"][i:i + 256] @ s["w"].T)
                                 for i in range(0, N, 256)])
    return s


# ------------------------------------------------------------------ plain forms
def _attn(s):
    c = s["case"]
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    G = Hq // Hkv
    out = torch.zeros_like(s["q"])
    start = 0
    for n in s["lens"]:
        q = s["q"][start:start + n].float().transpose(0, 1).reshape(Hkv, G, n, D)
        k = s["k"][start:start + n].float().permute(1, 2, 0)[:, None]      # [Hkv, 1, D, n]
        v = s["v"][start:start + n].float().transpose(0, 1)[:, None]       # [Hkv, 1, n, D]
        rows = max(1, min(n, 2 ** 28 // (Hq * n)))
        for i in range(0, n, rows):
            m = min(rows, n - i)
            end = i + m if c["causal"] else n
            x = (q[:, :, i:i + m] / math.sqrt(D)) @ k[..., :end]
            if c["causal"]:
                at = torch.arange(i, i + m, device=x.device)[:, None]
                key = torch.arange(end, device=x.device)
                hidden = key > at
                if c["window"] >= 0:
                    hidden = hidden | (key < at - c["window"])
                x = x.masked_fill(hidden, float("-inf"))
            w = (x - x.amax(-1, keepdim=True)).exp()
            o = (w @ v[..., :end, :]) / w.sum(-1, keepdim=True)
            out[start + i:start + i + m] = o.reshape(Hq, m, D).transpose(0, 1).to(out.dtype)
        start += n
    return out


def _places(s):
    """The sequence and the position of every packed row."""
    n = torch.diff(s["cu"]).long()
    seq = torch.repeat_interleave(torch.arange(len(n), device="cuda"), n)
    return seq, torch.arange(len(seq), device="cuda") - s["cu"].long()[seq]


def _rope(s):
    c = s["case"]
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    seq, at = _places(s)
    cos, sin = s["cos"][at].float()[:, None], s["sin"][at].float()[:, None]

    def turned(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
        half = torch.cat([-x[..., D // 2:], x[..., :D // 2]], -1)
        return (x * cos + half * sin).to(s["qkv"].dtype)

    x = s["qkv"].view(-1, Hq + 2 * Hkv, D)
    q, k = turned(x[:, :Hq], s["qn"]), turned(x[:, Hq:Hq + Hkv], s["kn"])
    if s["kc"] is None:
        return q, k
    if s["table"] is not None:
        seq, at = s["table"].long()[seq, at // BLOCK], at % BLOCK
    s["kc"][seq, :, at] = k
    s["vc"][seq, :, at] = x[:, Hq + Hkv:]
    return q, k, s["kc"], s["vc"]


def _first(x, value):
    """The lowest index of `value` in each row."""
    ix = torch.arange(x.shape[-1], device=x.device)
    return torch.where(x == value, ix, x.shape[-1]).amin(-1)


def _scores(x, tokens, temp, top):
    """Log probability and entropy of rows of logits in 32 bits; rank and alternatives."""
    t = x.gather(1, tokens[:, None])
    m = x.amax(-1, keepdim=True)
    d = (x - m) / temp
    w = d.exp()
    z = w.sum(-1, keepdim=True)
    lz = z.log()
    entropy = lz - torch.where(w > 0, w * d, 0).sum(-1, keepdim=True) / z
    rank = 1 + (x > t).sum(-1)
    vals, ids = [], []
    left = x.clone() if top else None
    for _ in range(top):
        best = left.amax(-1, keepdim=True)
        i = _first(left, best)
        left.scatter_(1, i[:, None], float("nan")).nan_to_num_(nan=float("-inf"))
        vals.append((best - m) / temp - lz)
        ids.append(i[:, None])
    none = x.new_empty(len(x), 0)
    return ((t - m) / temp - lz)[:, 0], entropy[:, 0], rank, torch.cat([none] + vals, 1), \
        torch.cat([none.long()] + ids, 1)


def _logprobs(s):
    c = s["case"]
    parts = [_scores(s["logits"][i:i + 512].float(), s["tokens"][i:i + 512], c["temp"], c["top"])
             for i in range(0, c["N"], 512)]
    return tuple(torch.cat(p) for p in zip(*parts))


def _head(s):
    c = s["case"]
    w = s["w"].float().T
    parts = [_scores(s["x"][i:i + 512].float() @ w, s["tokens"][i:i + 512], c["temp"], 0)[:2]
             for i in range(0, c["N"], 512)]
    return tuple(torch.cat(p) for p in zip(*parts))


# ------------------------------------------------------------------ the framework's
def _own(s):
    from torchplusplus_b200 import ops
    c = s["case"]
    if s["op"] == "attn":
        return ops.attention_packed(s["q"], s["k"], s["v"], s["cu"], causal=c["causal"],
                                    window_left=c["window"])
    if s["op"] == "rope":
        q, k = ops.qk_norm_rope_packed(s["qkv"], s["qn"], s["kn"], EPS, s["cos"], s["sin"],
                                       s["cu"], c["Hq"], c["Hkv"], k_cache=s["kc"],
                                       v_cache=s["vc"], block_table=s["table"])
        return (q, k) if s["kc"] is None else (q, k, s["kc"], s["vc"])
    if s["op"] == "logprobs":
        return ops.token_logprobs(s["logits"], s["tokens"], temperature=c["temp"], top=c["top"])
    return ops.linear_logprobs(s["x"], s["w"], s["tokens"], temperature=c["temp"])


def run(state):
    if own:
        return _own(state)
    return {"attn": _attn, "rope": _rope, "logprobs": _logprobs, "head": _head}[state["op"]](state)


# ------------------------------------------------------------------ work
def work(case):
    c = case
    if c["op"] in ("attn", "rope"):
        Hq, Hkv, D, lens = c["Hq"], c["Hkv"], c["D"], lengths(c)
        N = sum(lens)
        if c["op"] == "rope":
            rows = Hq + 2 * Hkv + Hq + Hkv + (2 * Hkv if c["cache"] != "none" else 0)
            return dict(bytes=2.0 * N * rows * D + 4 * max(lens) * D,
                        flops=8.0 * N * (Hq + Hkv) * D)
        pairs = 0
        for n in lens:
            if not c["causal"]:
                pairs += n * n
            else:
                w = n if c["window"] < 0 else min(n, c["window"] + 1)
                pairs += w * (w + 1) // 2 + (n - w) * w
        return dict(bytes=4.0 * N * (Hq + Hkv) * D, flops=4.0 * pairs * Hq * D)
    N, V = c["N"], c["V"]
    if c["op"] == "logprobs":
        size = 4 if c["dtype"] == "f32" else 2
        return dict(bytes=float(size) * N * V + N * (24 + 12 * c["top"]), flops=6.0 * N * V)
    return dict(bytes=2.0 * (N + V) * c["E"] + 16 * N, flops=2.0 * N * V * c["E"])


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The outputs from the definitions in 64 bits, one head or some rows at a time."""
    s, c = prepare(case, seed), case
    if c["op"] == "attn":
        Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        for a, b in zip(s["cu"].tolist()[:-1], s["cu"].tolist()[1:]):
            for h in range(Hq):
                q = s["q"][a:b, h].double() * D ** -0.5
                k = s["k"][a:b, h // (Hq // Hkv)].double()
                v = s["v"][a:b, h // (Hq // Hkv)].double()
                for i in range(0, b - a, 4096):
                    lo, hi = 0, b - a
                    if c["causal"]:
                        hi = min(hi, i + 4096)
                    if c["causal"] and c["window"] >= 0:
                        lo = max(0, i - c["window"])
                    x = q[i:i + 4096] @ k[lo:hi].T
                    if c["causal"]:
                        far = torch.arange(i, i + len(x), device="cuda")[:, None] \
                            - torch.arange(lo, hi, device="cuda")
                        x[far < 0] = float("-inf")
                        if c["window"] >= 0:
                            x[far > c["window"]] = float("-inf")
                    out[a + i:a + i + len(x), h] = torch.softmax(x, 1) @ v[lo:hi]
        return out
    if c["op"] == "rope":
        Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
        x = s["qkv"].double().view(-1, Hq + 2 * Hkv, D)
        at = torch.cat([torch.arange(n, device="cuda") for n in s["lens"]])
        cos, sin = (t.double()[at][:, None, :D // 2] for t in (s["cos"], s["sin"]))
        out = []
        for part, w in ((x[:, :Hq], s["qn"]), (x[:, Hq:Hq + Hkv], s["kn"])):
            if w is not None:
                part = part * w.double() / (part.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
            a, b = part[..., :D // 2], part[..., D // 2:]
            out.append(torch.cat([a * cos - b * sin, b * cos + a * sin], -1))
        if s["kc"] is None:
            return tuple(out)
        kc, vc = s["kc"].double(), s["vc"].double()
        a = 0
        for b, n in enumerate(s["lens"]):
            for j in range(0, n, BLOCK):
                m = min(BLOCK, n - j)
                for cache, new in ((kc, out[1]), (vc, x[:, Hq + Hkv:])):
                    rows = new[a + j:a + j + m].transpose(0, 1)
                    if s["table"] is None:
                        cache[b, :, j:j + m] = rows
                    else:
                        cache[int(s["table"][b, j // BLOCK]), :, :m] = rows
            a += n
        return out[0], out[1], kc, vc
    lp, ent, rank, best = [], [], [], []
    for i in range(0, c["N"], 256):
        t = s["tokens"][i:i + 256, None]
        if c["op"] == "head":
            x = s["x"][i:i + 256].double() @ s["w"].double().T
        else:
            x = s["logits"][i:i + 256].double()
            rank.append((x >= x.gather(1, t)).sum(1) - (x == x.gather(1, t)).sum(1) + 1)
        l = torch.log_softmax(x / c["temp"], 1)
        lp.append(l.gather(1, t)[:, 0])
        ent.append(-(l.exp() * l).sum(1))
        if c["op"] == "logprobs":
            best.append(l.topk(c["top"], 1).values)
    if c["op"] == "head":
        return torch.cat(lp), torch.cat(ent)
    return torch.cat(lp), torch.cat(ent), torch.cat(rank), torch.cat(best), None
