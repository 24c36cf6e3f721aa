"""Cases of the draft-tree operators: attention of a tree of drafted tokens over
a KV cache, its q/k norm and rotary positions, the verification of the tree
against the target's logits, and the commit of the accepted path's K/V.

`run` computes an operator in its plain form (elementary torch operations in 32
bits) or, where `own` is true, by the framework's entry points."""
import math

import torch

own = False

HALF = {"bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 64  # keys in a block of the paged cache
EPS = 1e-6


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one chat of a few hundred tokens, five drafted tokens: latency is all
        dict(name="attn 1x5 ctx 130", op="attn", B=1, T=5, ctx=130, Hq=16, Hkv=8, D=128,
             dtype="bf16", paged=False, window=-1, ragged=False),
        # one long conversation with a wide tree
        dict(name="attn 1x64 ctx 8191", op="attn", B=1, T=64, ctx=8191, Hq=16, Hkv=8, D=128,
             dtype="bf16", paged=False, window=-1, ragged=False),
        # the serving batch of the decode benchmark, a small tree a sequence
        dict(name="attn 32x8 ctx 640", op="attn", B=32, T=8, ctx=640, Hq=16, Hkv=8, D=128,
             dtype="bf16", paged=False, window=-1, ragged=True),
        # many sequences of very different lengths in a paged cache
        dict(name="attn 64x13 ctx 4096 paged", op="attn", B=64, T=13, ctx=4096, Hq=32, Hkv=8,
             D=128, dtype="f16", paged=True, window=-1, ragged=True),
        # few very long contexts with wide trees: the most work of the set
        dict(name="attn 4x64 ctx 32768", op="attn", B=4, T=64, ctx=32768, Hq=16, Hkv=8, D=128,
             dtype="bf16", paged=False, window=-1, ragged=False),
        # a single sequence's draft chain with its draft model's logits
        dict(name="verify 1x5 chain", op="verify", B=1, T=5, V=151936, dtype="bf16", chain=True,
             draft=True, temp=1.0),
        # a serving batch with trees of top tokens (no draft distribution)
        dict(name="verify 32x32 tree", op="verify", B=32, T=32, V=151936, dtype="bf16",
             chain=False, draft=False, temp=0.8),
        # many sequences, longer chains, a small vocabulary of odd size
        dict(name="verify 64x9 chain odd", op="verify", B=64, T=9, V=32003, dtype="f16",
             chain=True, draft=True, temp=1.0),
        # the accepted path of one sequence, all layers of the benchmark model
        dict(name="commit 28x1x8", op="commit", L=28, B=1, T=8, Hkv=8, D=128, cap=1024,
             dtype="bf16", paged=False),
        # the same for a serving batch over a paged cache
        dict(name="commit 28x64x16 paged", op="commit", L=28, B=64, T=16, Hkv=8, D=128, cap=256,
             dtype="f16", paged=True),
        # q/k norm and rotary positions of one small tree
        dict(name="rope 1x8", op="rope", B=1, T=8, Hq=16, Hkv=8, D=128, ctx=2048, dtype="bf16",
             norm=True),
        # and of wide trees of a serving batch
        dict(name="rope 64x64", op="rope", B=64, T=64, Hq=32, Hkv=8, D=128, ctx=8192,
             dtype="f16", norm=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "verify", "verify", "commit", "rope"])
    dtype = rng.choice(["bf16", "f16"])
    Hq, Hkv = rng.choice([(16, 8), (32, 8), (16, 16), (8, 1), (12, 4), (28, 4)])
    D = rng.choice([64, 128, 128])
    if op == "attn":
        T = _log(rng, 1, 128)
        B = _log(rng, 1, 64)
        # no more bytes of cache, and no more products, than the largest listed case
        most = 4 * 8 * 32768 * 128
        ctx = _log(rng, 1, 32768)
        ctx = max(0, min(ctx, most // (B * Hkv * D), most * 128 // (B * T * Hq * D)) - 1)
        return dict(op=op, B=B, T=T, ctx=ctx, Hq=Hq, Hkv=Hkv, D=D, dtype=dtype,
                    paged=rng.random() < 0.5, window=rng.choice([-1, -1, _log(rng, 16, 4096)]),
                    ragged=rng.random() < 0.7)
    if op == "verify":
        chain = rng.random() < 0.5
        T = _log(rng, 1, 16) if chain else _log(rng, 2, 64)
        V = _log(rng, 1000, 151936)
        draft = rng.random() < (0.7 if chain else 0.3)
        B = min(_log(rng, 1, 64), max(1, 32 * 32 * 151936 // (V * T * (2 if draft else 1))))
        return dict(op=op, B=B, T=T, V=V, dtype=dtype, chain=chain, draft=draft,
                    temp=rng.choice([0.0, 0.6, 1.0]))
    if op == "commit":
        return dict(op=op, L=_log(rng, 1, 28), B=_log(rng, 1, 64), T=_log(rng, 1, 64), Hkv=Hkv,
                    D=D, cap=rng.choice([192, 256]), dtype=dtype, paged=rng.random() < 0.5)
    return dict(op=op, B=_log(rng, 1, 64), T=_log(rng, 1, 64), Hq=Hq, Hkv=Hkv, D=D,
                ctx=_log(rng, 1, 8192), dtype=dtype, norm=rng.random() < 0.7)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rand(g, *shape, dtype=torch.float32):
    return torch.rand(shape, generator=g, device="cuda").to(dtype)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _trees(g, B, T, chain):
    """Parents (int32 [B, T], -1 at the root, a parent before its children):
    a chain, or trees whose later nodes hang from the middle of those before."""
    i = torch.arange(T, device="cuda")
    if chain:
        par = (i - 1).expand(B, T)
    else:
        par = (_rand(g, B, T).sqrt() * i * 0.8).long()
        par[:, 0] = -1
    return par.to(torch.int32).contiguous()


def _ancestors(par):
    """bool [B, T, T]: node i sees node j (its ancestors and itself)."""
    B, T = par.shape
    anc = torch.zeros(B, T, T, dtype=torch.bool, device=par.device)
    b = torch.arange(B, device=par.device)
    for i in range(T):
        if i:
            anc[:, i] = anc[b, par[:, i].long()]
        anc[:, i, i] = True
    return anc


def _pack(see):
    """bool [B, T, T] -> int64 [B, T, ceil(T / 64)], bit j % 64 of word j // 64."""
    B, T, _ = see.shape
    W = (T + 63) // 64
    bits = torch.zeros(B, T, W * 64, dtype=torch.int64, device=see.device)
    bits[..., :T] = see
    return (bits.view(B, T, W, 64) << torch.arange(64, device=see.device)).sum(-1)


def _unpack(mask, T):
    j = torch.arange(T, device=mask.device)
    return ((mask[..., j // 64] >> (j % 64)) & 1).bool()


def _lengths(g, B, ctx, ragged):
    if not ragged or ctx == 0:
        return torch.full((B,), ctx, dtype=torch.int32, device="cuda")
    return (ctx - (_rand(g, B) * (0.6 * ctx)).long()).to(torch.int32)


def _blocks(g, B, n):
    """A block table [B, n] of shuffled blocks, and their number."""
    return torch.randperm(B * n, generator=g, device="cuda").view(B, n).to(torch.int32), B * n


def prepare(case, seed):
    g, c = _gen(seed), case
    s = dict(case=c, op=c["op"])
    dt = HALF[c["dtype"]]
    B, T = c["B"], c["T"]
    if c["op"] == "attn":
        Hkv, D = c["Hkv"], c["D"]
        s["q"] = 2.5 * _randn(g, B, T, c["Hq"], D, dtype=dt)  # scores that prefer some keys
        s["kt"] = _randn(g, B, T, Hkv, D, dtype=dt)
        s["vt"] = _randn(g, B, T, Hkv, D, dtype=dt)
        s["mask"] = _pack(_ancestors(_trees(g, B, T, False)))
        s["ctx"] = _lengths(g, B, c["ctx"], c["ragged"])
        if c["paged"]:
            n = max(1, -(-c["ctx"] // BLOCK))
            s["table"], nb = _blocks(g, B, n)
            s["k"] = _randn(g, nb, Hkv, BLOCK, D, dtype=dt)
            s["v"] = _randn(g, nb, Hkv, BLOCK, D, dtype=dt)
        else:
            s["k"] = _randn(g, B, Hkv, max(1, c["ctx"]), D, dtype=dt)
            s["v"] = _randn(g, B, Hkv, max(1, c["ctx"]), D, dtype=dt)
    elif c["op"] == "verify":
        V = c["V"]
        # a target with a few likely tokens and a long tail, and a draft near it
        logits = _randn(g, B, T, V, dtype=dt) * 2.5
        s["par"] = _trees(g, B, T, c["chain"])
        s["logits"] = logits
        s["u"] = _rand(g, B, T)
        tokens = torch.zeros(B, T, dtype=torch.int64, device="cuda")
        s["draft"] = None
        b = torch.arange(B, device="cuda")
        if c["draft"]:
            s["draft"] = (logits + 0.6 * _randn(g, B, T, V, dtype=dt))
            for i in range(1, T):  # drawn from the draft, by the largest of noise + logit
                x = s["draft"][b, s["par"][:, i].long()].float() / (c["temp"] or 1.0)
                tokens[:, i] = (x - (-_rand(g, B, V).clamp_min(1e-30).log()).log()).argmax(-1)
        else:
            best = logits.topk(8, -1).indices
            nth = torch.zeros(B, T, dtype=torch.int64, device="cuda")  # children so far
            for i in range(1, T):
                p = s["par"][:, i].long()
                tokens[:, i] = best[b, p, nth[b, p].clamp_max(7)]
                nth[b, p] += 1
        s["tokens"] = tokens
    elif c["op"] == "commit":
        L, Hkv, D, cap = c["L"], c["Hkv"], c["D"], c["cap"]
        s["kt"] = _randn(g, L, B, T, Hkv, D, dtype=dt)
        s["vt"] = _randn(g, L, B, T, Hkv, D, dtype=dt)
        count = 1 + (_rand(g, B) * min(T, 8)).long()
        order = _rand(g, B, T)
        order[:, 0] = -1                                      # a path begins at the root
        order = order.argsort(-1)
        order = torch.where(torch.arange(T, device="cuda") < count[:, None], order, T).sort(-1)[0]
        s["path"] = torch.where(order < T, order, -1).to(torch.int32)
        s["count"] = count.to(torch.int32)
        s["ctx"] = (_rand(g, B) * (cap - T)).to(torch.int32)
        s["table"] = None
        if c["paged"]:
            s["table"], nb = _blocks(g, B, cap // BLOCK)
            shape = (L, nb, Hkv, BLOCK, D)
        else:
            shape = (L, B, Hkv, cap, D)
        s["k"], s["v"] = _randn(g, *shape, dtype=dt), _randn(g, *shape, dtype=dt)
    else:
        Hq, Hkv, D, ctx = c["Hq"], c["Hkv"], c["D"], c["ctx"]
        s["qkv"] = _randn(g, B, T, (Hq + 2 * Hkv) * D, dtype=dt)
        s["qn"] = s["kn"] = None
        if c["norm"]:
            s["qn"] = (1 + 0.1 * _randn(g, D)).to(dt)
            s["kn"] = (1 + 0.1 * _randn(g, D)).to(dt)
        depth = _ancestors(_trees(g, B, T, False)).sum(-1) - 1
        s["pos"] = ((_rand(g, B, 1) * ctx).long() + depth).to(torch.int32)
        inv = 1e6 ** (-torch.arange(0, D, 2, device="cuda") / D)
        ang = torch.arange(ctx + T, device="cuda")[:, None] * inv
        ang = torch.cat([ang, ang], 1)
        s["cos"], s["sin"] = ang.cos().half(), ang.sin().half()
    return s


# ------------------------------------------------------------------ plain forms
def _context(s, x, paged):
    """The cache's rows [B, Hkv, n, D] of each sequence, in 32 bits."""
    if not paged:
        return x.float()
    B, n = s["table"].shape
    y = x[s["table"].long()]                       # [B, n, Hkv, BLOCK, D]
    return y.permute(0, 2, 1, 3, 4).reshape(B, y.shape[2], n * BLOCK, -1).float()


def _visible(s, n, T):
    """bool [B, T, n + T]: which of n cache rows and T nodes each node sees."""
    c = s["case"]
    see = _unpack(s["mask"], T)
    key = torch.arange(n, device="cuda")
    old = (key < s["ctx"][:, None, None]).expand(-1, T, -1)
    if c["window"] >= 0:
        at = s["ctx"][:, None] + see.sum(-1) - 1   # a node's own position
        old = old & (key >= (at - c["window"])[..., None])
    return torch.cat([old, see], -1)


def _attn(s):
    c = s["case"]
    B, T, Hq, Hkv, D = c["B"], c["T"], c["Hq"], c["Hkv"], c["D"]
    k = torch.cat([_context(s, s["k"], c["paged"]), s["kt"].float().transpose(1, 2)], 2)
    v = torch.cat([_context(s, s["v"], c["paged"]), s["vt"].float().transpose(1, 2)], 2)
    see = _visible(s, k.shape[2] - T, T)[:, None, None]          # [B, 1, 1, T, N]
    q = s["q"].float().permute(0, 2, 1, 3).reshape(B, Hkv, Hq // Hkv * T, D)
    x = (q @ k.transpose(2, 3) / math.sqrt(D)).view(B, Hkv, Hq // Hkv, T, -1)
    x = x.masked_fill(~see, float("-inf"))
    m = x.amax(-1, keepdim=True)
    w = torch.where(see, (x - torch.where(m.isinf(), 0, m)).exp(), 0)
    z = w.sum(-1, keepdim=True)
    w = torch.where(z > 0, w / z, 0).view(B, Hkv, -1, k.shape[2])
    o = (w @ v).view(B, Hq, T, D).transpose(1, 2)
    return o.to(s["q"].dtype)


FIX = 2.0 ** 40  # weights are summed as whole multiples of 1 / FIX: exact in any order


def _weights(row, temp):
    """exp((l - max) / temp) over the last axis in 32 bits, 0 at NaN."""
    x = row.float()
    m = torch.where(x.isnan(), float("-inf"), x).amax(-1, keepdim=True)
    w = ((x - m) * torch.tensor(1.0 / temp, dtype=torch.float32, device=x.device)).exp()
    return torch.where(w.isnan(), 0, w)


def _fixed(w):
    return (w.double() * FIX).round().long()


def _share(w):
    """w over its sum (0 where the sum is 0)."""
    z = (_fixed(w).sum(-1, keepdim=True).double() / FIX).float()
    return torch.where(z > 0, w / z, 0)


def _verify(s):
    """Walks every tree from its root: a child is accepted with its share of
    what is left of the target's distribution (over the draft's, where given),
    and the next token is drawn from what is left at the last accepted node."""
    c, tokens, par, u = s["case"], s["tokens"], s["par"], s["u"]
    B, T = tokens.shape
    b = torch.arange(B, device="cuda")
    cur = torch.zeros(B, dtype=torch.int64, device="cuda")
    path = torch.full((B, T), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = 0
    count = torch.ones(B, dtype=torch.int64, device="cuda")

    def left(node):
        row = s["logits"][b, node]
        if c["temp"] == 0:
            x = torch.where(row.isnan(), float("-inf"), row.float())
            top = x.amax(-1, keepdim=True)
            ix = torch.arange(x.shape[-1], device="cuda")
            first = torch.where(x == top, ix, x.shape[-1]).amin(-1, keepdim=True)
            return ((ix == first) & (top > float("-inf"))).float()
        w = _weights(row, c["temp"])
        return w if s["draft"] is None else _share(w)

    def drafted(node):
        return _share(_weights(s["draft"][b, node], c["temp"]))

    greedy = c["temp"] == 0
    with_q = s["draft"] is not None and not greedy
    p = left(cur)
    q = drafted(cur) if with_q else None
    for i in range(1, T):
        t = tokens[:, i]
        try_ = par[:, i] == cur
        if with_q:
            ok = u[:, i] * q[b, t] < p[b, t]
            r = (p - q).clamp_min(0)
            z = (_fixed(r).sum(-1, keepdim=True).double() / FIX).float()
            r = torch.where(z > 0, r / z, p)
        else:
            w = _fixed(p)
            z = w.sum(-1).double()
            ok = u[:, i].double() * z < w[b, t].double() if not greedy else w[b, t] > 0
            r = p.clone()
            r[b, t] = 0
            if greedy:
                r = p
        take = try_ & ok
        p = torch.where((try_ & ~ok)[:, None], r, p)
        path[b, count.clamp_max(T - 1)] = torch.where(take, i, path[b, count.clamp_max(T - 1)]).to(torch.int32)
        count += take
        cur = torch.where(take, i, cur)
        p = torch.where(take[:, None], left(cur), p)
        if with_q:
            q = torch.where(take[:, None], drafted(cur), q)
    w = _fixed(p)
    cum = w.cumsum(-1)
    z = cum[:, -1:]
    at = torch.minimum((u[:, :1].double() * z.double()).floor().long(), z - 1)
    nxt = (cum <= at).sum(-1)
    return path, count.to(torch.int32), torch.where(z[:, 0] > 0, nxt, -1)


def _commit(s):
    T, cap = s["case"]["T"], s["case"]["cap"]
    b, i = torch.nonzero(torch.arange(T, device="cuda") < s["count"][:, None], as_tuple=True)
    row = s["ctx"].long()[b] + i
    node = s["path"].long()[b, i]
    if s["table"] is None:
        s["k"][:, b, :, row] = s["kt"][:, b, node].transpose(0, 1)
        s["v"][:, b, :, row] = s["vt"][:, b, node].transpose(0, 1)
    else:
        blk = s["table"].long()[b, row // BLOCK]
        s["k"][:, blk, :, row % BLOCK] = s["kt"][:, b, node].transpose(0, 1)
        s["v"][:, blk, :, row % BLOCK] = s["vt"][:, b, node].transpose(0, 1)
    return s["k"], s["v"]


def _rope(s):
    c = s["case"]
    B, T, Hq, Hkv, D = c["B"], c["T"], c["Hq"], c["Hkv"], c["D"]
    at = s["pos"].long()
    cos, sin = s["cos"][at].float()[:, :, None], s["sin"][at].float()[:, :, None]

    def turned(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
        half = torch.cat([-x[..., D // 2:], x[..., :D // 2]], -1)
        return (x * cos + half * sin).to(s["qkv"].dtype)

    x = s["qkv"].view(B, T, Hq + 2 * Hkv, D)
    return turned(x[:, :, :Hq], s["qn"]), turned(x[:, :, Hq:Hq + Hkv], s["kn"])


# ------------------------------------------------------------------ the framework's
def _own(s):
    from torchplusplus_b200 import ops
    c = s["case"]
    if s["op"] == "attn":
        if c["paged"]:
            return ops.attention_tree_paged(s["q"], s["k"], s["v"], s["table"], s["kt"], s["vt"],
                                            s["ctx"], c["ctx"], s["mask"],
                                            window_left=c["window"])
        return ops.attention_tree(s["q"], s["k"], s["v"], s["kt"], s["vt"], s["ctx"], c["ctx"],
                                  s["mask"], window_left=c["window"])
    if s["op"] == "verify":
        return ops.verify_tree(s["logits"], s["tokens"], s["par"], s["u"],
                               temperature=c["temp"], draft_logits=s["draft"])
    if s["op"] == "commit":
        ops.kv_commit(s["kt"], s["vt"], s["path"], s["count"], s["ctx"], s["k"], s["v"],
                      block_table=s["table"])
        return s["k"], s["v"]
    return ops.qk_norm_rope_tree(s["qkv"], s["qn"], s["kn"], EPS, s["cos"], s["sin"], s["pos"],
                                 c["Hq"], c["Hkv"])


def run(state):
    if own:
        return _own(state)
    return {"attn": _attn, "verify": _verify, "commit": _commit, "rope": _rope}[state["op"]](state)


# ------------------------------------------------------------------ work
def work(case):
    c = case
    B, T = c["B"], c["T"]
    if c["op"] == "attn":
        Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
        n = c["ctx"] * (0.7 if c["ragged"] else 1.0)       # mean length of a context
        if c["window"] >= 0:
            n = min(n, c["window"] + 1)
        by = 2 * B * (2 * n * Hkv * D + 2 * T * Hkv * D + 2 * T * Hq * D) + B * T * 8 * -(-T // 64)
        return dict(bytes=by, flops=4.0 * B * T * Hq * D * (n + T / 4))
    if c["op"] == "verify":
        # the rows of the accepted path: about three quarters of the tests pass
        depth = T - 1 if c["chain"] else math.log2(T)
        rows = (1 - 0.75 ** (depth + 1)) / 0.25
        if c["draft"] and c["temp"] > 0:
            rows += min(1.0, depth)                          # the draft's where a test fails
        return dict(bytes=2.0 * B * rows * c["V"] + B * T * 20, flops=8.0 * B * rows * c["V"])
    if c["op"] == "commit":
        kept = B * (1 + (min(T, 8) - 1) / 2)
        return dict(bytes=8.0 * kept * c["L"] * c["Hkv"] * c["D"] + B * (T + 2) * 4, flops=0)
    n = B * T * (c["Hq"] + c["Hkv"]) * c["D"]
    return dict(bytes=4.0 * n + B * T * (4 + 4 * c["D"]), flops=8.0 * n)


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The outputs from the definitions, one head or token row at a time."""
    s, c = prepare(case, seed), case
    if c["op"] == "verify":
        return None  # whole numbers
    if c["op"] == "commit":
        out = [s["k"].double(), s["v"].double()]
        for b, n in enumerate(s["count"].tolist()):
            for i, node in enumerate(s["path"][b, :n].tolist()):
                row = int(s["ctx"][b]) + i
                for x, new in zip(out, (s["kt"], s["vt"])):
                    if c["paged"]:
                        x[:, int(s["table"][b, row // BLOCK]), :, row % BLOCK] = new[:, b, node].double()
                    else:
                        x[:, b, :, row] = new[:, b, node].double()
        return tuple(out)
    B, T, Hq, Hkv, D = c["B"], c["T"], c["Hq"], c["Hkv"], c["D"]
    if c["op"] == "attn":
        out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device="cuda")
        bits = s["mask"].cpu().tolist()
        for b in range(B):
            n = int(s["ctx"][b])
            see = torch.tensor([[(r[j // 64] >> (j % 64)) & 1 for j in range(T)] for r in bits[b]],
                               dtype=torch.bool, device="cuda")
            if c["paged"]:
                rows = [x[s["table"][b].long()].transpose(1, 2).reshape(-1, Hkv, D)[:n]
                        for x in (s["k"], s["v"])]
            else:
                rows = [x[b, :, :n].transpose(0, 1) for x in (s["k"], s["v"])]
            k = torch.cat([rows[0], s["kt"][b]]).double()
            v = torch.cat([rows[1], s["vt"][b]]).double()
            place = torch.arange(n, device="cuda").expand(T, n)
            old = torch.ones(T, n, dtype=torch.bool, device="cuda")
            if c["window"] >= 0:
                old = n + see.sum(1, keepdim=True) - 1 - place <= c["window"]
            bias = torch.zeros(T, n + T, dtype=torch.float64, device="cuda")
            bias[~torch.cat([old, see], 1)] = float("-inf")
            for h in range(Hq):
                x = s["q"][b, :, h].double() @ k[:, h // (Hq // Hkv)].T * D ** -0.5 + bias
                out[b, :, h] = torch.softmax(x, 1) @ v[:, h // (Hq // Hkv)]
        return out
    out = []
    x = s["qkv"].double().view(B, T, Hq + 2 * Hkv, D)
    for part, w in ((x[:, :, :Hq], s["qn"]), (x[:, :, Hq:Hq + Hkv], s["kn"])):
        if w is not None:
            part = part * w.double() / (part.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
        a, b = part[..., :D // 2], part[..., D // 2:]
        cos = s["cos"].double()[s["pos"].long()][:, :, None, :D // 2]
        sin = s["sin"].double()[s["pos"].long()][:, :, None, :D // 2]
        out.append(torch.cat([a * cos - b * sin, b * cos + a * sin], -1))
    return tuple(out)
