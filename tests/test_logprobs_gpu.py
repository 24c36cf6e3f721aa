"""Log probabilities of given tokens, from logits and from the LM head's operands,
against the definitions in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def oracle(x, tokens, temperature, top):
    """The five outputs in 64 bits."""
    N, V = x.shape
    y = x.double() / temperature
    m = y.amax(1, keepdim=True)
    w = (y - torch.where(m == -math.inf, 0, m)).exp()
    z = w.sum(1, keepdim=True)
    l = y - torch.where(m == -math.inf, 0, m) - z.log()
    broken = (x.isnan() | (x == math.inf)).any(1)
    none = (z == 0)[:, 0] & ~broken
    l[none] = -math.inf
    l[broken] = math.nan
    ent = -torch.where(l == -math.inf, 0, l.exp() * l).sum(1)
    has = (tokens >= 0) & (tokens < V)
    t = tokens.clamp(0, V - 1)[:, None]
    lp = torch.where(has, l.gather(1, t)[:, 0], 0)
    tv = x.gather(1, t)
    above = (x > tv) | (x.isnan() & ~tv.isnan())
    above &= ~tv.isnan()
    rank = torch.where(has, 1 + above.sum(1), 0)
    if top == 0:
        return lp, ent, rank, x.new_empty(N, 0).double(), tokens.new_empty(N, 0)
    # stable (ties by id; -0 + 0 is 0), with NaN before +inf: two sorts
    key = torch.where(x.isnan(), math.inf, x.double()) + 0.0
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices
    nan = x.isnan().gather(1, ids).to(torch.int8)
    ids = ids.gather(1, torch.sort(nan, dim=1, descending=True, stable=True).indices)[:, :top]
    return lp, ent, rank, l.gather(1, ids), ids


def same(got, ref, tol):
    ok = (got.double() - ref).abs() <= tol
    # infinite in both, or beyond the largest float32 (3.4e38), which rounds to infinity
    ok |= (got == ref.float()) | (got.isnan() & ref.isnan())
    assert ok.all(), ((got.double() - ref).abs() / tol).nan_to_num().max().item()


def check(x, tokens, temperature=1.0, top=0):
    """Tolerance: y = (x - m) / T is off by 2 roundings (2^-23 |y|), a weight by that and the
    exponential's 2^-22 besides 2^-23 a sum's step over at most 16 steps of nesting; log and the last product
    round twice more.  |y| of what weighs anything is at most 104 (the rest is 0 in both)."""
    from torchplusplus_b200 import ops
    got = ops.token_logprobs(x, tokens, temperature=temperature, top=top)
    ref = oracle(x, tokens, temperature, top)
    assert got[0].dtype == F32 and got[1].dtype == F32
    eps = (104 + 2 ** 7) * 2.0 ** -23
    V = x.shape[1]
    rel = 2.0 ** -22
    same(got[0], ref[0], eps + rel * ref[0].abs())
    same(got[1], ref[1], (2 * math.log(V) + 2) * eps + rel * ref[1].abs())
    assert torch.equal(got[2], ref[2])
    assert torch.equal(got[4], ref[4])
    same(got[3], ref[3], eps + rel * ref[3].abs())


def logits(seed, N, V, dtype, spread=3.0):
    return (torch.randn(N, V, generator=gen(seed), device="cuda") * spread).to(dtype)


def tokens_for(seed, N, V):
    return torch.randint(0, V, (N,), generator=gen(seed + 1000), device="cuda")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("N,V", [(1, 1), (3, 7), (1, 8), (40, 33), (5, 1000), (2, 4096), (300, 2049),
                                 (1, 32003), (9, 32003), (500, 5003), (2, 151936), (70, 20000)])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_token_logprobs(dtype, N, V, top):
    check(logits(V, N, V, dtype), tokens_for(N, N, V), top=min(top, V))


@pytest.mark.parametrize("temperature", [0.05, 0.6, 3.0])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_temperatures(temperature, dtype):
    check(logits(1, 33, 3001, dtype), tokens_for(1, 33, 3001), temperature, 4)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("off,ld", [(0, 1008), (3, 1013), (1, 1001)])
def test_strided_rows(dtype, off, ld):
    room = logits(2, 20, ld, dtype)
    check(room[:, off:off + 1000], tokens_for(2, 20, 1000), top=6)
    wide = logits(3, 1000, 20, dtype).T                     # columns apart: copied
    check(wide, tokens_for(3, 20, 1000), top=6)


@pytest.mark.parametrize("N", [2, 600])
@pytest.mark.parametrize("V", [100, 30011])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_that_are_odd(N, V, dtype):
    """Ties in number, order against the search, masks of -inf and of the type's lowest value,
    rows of nothing, infinities, NaN."""
    low, ix = torch.finfo(dtype).min, torch.arange(V, device="cuda")
    rows = [
        torch.zeros(V),                                                    # all equal
        ix / V * 60 - 30, 30 - ix / V * 60,                                # in order
        torch.where(ix % 3 == 0, -math.inf, torch.where(ix % 37 == 5, 1.0, 0.0)),
        torch.where(ix < 3, -ix.float(), -math.inf),                       # three tokens left
        torch.where(ix < V - 2, -math.inf, 2.0),
        torch.where(ix < 5, 3.0 * (ix % 2), low),
        torch.full((V,), low),                                             # uniform
        torch.full((V,), -math.inf),                                       # nothing
        torch.where(ix == V // 2, math.nan, ix % 11),
        torch.where(ix == V - 1, math.inf, ix % 11),
        torch.full((V,), math.nan),
        torch.where((ix == 0) | (ix == 8), math.nan, torch.where(ix == 4, math.inf, ix % 5)),
        torch.where(ix % 2 == 0, 0.0, -0.0),
        torch.where(ix == V - 1, math.nan, -math.inf),
        torch.where(ix == V - 1, 60.0, ix % 13),                           # one token, at the end
        torch.where(ix % 8 == 7, 5.0, 4.0),
    ]
    rows = [r.to(device="cuda", dtype=dtype) for r in rows]
    if N > len(rows):
        batches = [logits(4, N, V, dtype)]
        for i, r in enumerate(rows):
            batches[0][i], batches[0][i * 31 + 20] = r, r
    else:
        batches = [torch.stack(rows[i:i + N]) for i in range(0, len(rows), N)]
    for x in batches:
        tok = tokens_for(4, len(x), V)
        for top in (0, 1, 9, 32):
            check(x, tok, top=top)


def test_lowest_mask_with_a_high_row():
    """Differences that overflow 32 bits weigh nothing."""
    x = torch.full((3, 500), torch.finfo(F32).min, device="cuda")
    x[0, 7] = 3e38
    x[1, 100:104] = 1e38
    x[2, 499] = -1.0
    check(x, torch.tensor([7, 3, 499], device="cuda"), top=3)


def test_tokens_outside_the_vocabulary():
    from torchplusplus_b200 import ops
    x = logits(6, 4, 999, BF16)
    tok = torch.tensor([-1, 999, 5, 1 << 40], device="cuda")
    check(x, tok, top=3)
    lp, _, rank, _, _ = ops.token_logprobs(x, tok)
    assert lp[[0, 1, 3]].eq(0).all() and rank[[0, 1, 3]].eq(0).all() and rank[2] > 0


def test_no_rows_and_a_graph():
    from torchplusplus_b200 import ops
    out = ops.token_logprobs(logits(7, 0, 50, BF16), tokens_for(7, 0, 50), top=3)
    assert [tuple(t.shape) for t in out] == [(0,), (0,), (0,), (0, 3), (0, 3)]
    x, tok = logits(8, 5, 9000, BF16), tokens_for(8, 5, 9000)
    w = (torch.randn(3001, 64, generator=gen(9), device="cuda")).to(BF16)
    h = (torch.randn(5, 64, generator=gen(10), device="cuda")).to(BF16)
    ops.token_logprobs(x, tok, top=2), ops.linear_logprobs(h, w, tok % 3001)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a = ops.token_logprobs(x, tok, top=2)
        b = ops.linear_logprobs(h, w, tok % 3001)
    x.copy_(logits(11, 5, 9000, BF16))
    h.mul_(0.5)
    g.replay()
    for got, want in zip(a + b, ops.token_logprobs(x, tok, top=2) + ops.linear_logprobs(h, w, tok % 3001)):
        assert torch.equal(got, want)


# ------------------------------------------------------------------ from the head
def check_head(x, w, tokens, temperature=1.0):
    """Tolerance: a logit is a sum of E exact products in 32 bits, whatever their order and rounding
    off by at most E 2^-23 of the sum of their magnitudes; log softmax moves by at most twice that
    (over T), the entropy by 2 ln V + 2 times; and as for logits that are given."""
    from torchplusplus_b200 import ops
    got = ops.linear_logprobs(x, w, tokens, temperature=temperature)
    N, E = x.shape
    V = w.shape[0]
    y = x.double() @ w.double().T
    ref = oracle(y, tokens, temperature, 0)
    d = E * 2.0 ** -23 * (x.double().abs() @ w.double().abs().T).amax(1) / temperature
    eps = (104 + 2 ** 7) * 2.0 ** -23
    same(got[0], ref[0], 2 * d + eps + 2.0 ** -22 * ref[0].abs())
    same(got[1], ref[1], (2 * math.log(V) + 2) * (d + eps) + 2.0 ** -22 * ref[1].abs())


def operands(seed, N, E, V, dtype):
    g = gen(seed)
    x = torch.randn(N, E, generator=g, device="cuda").to(dtype)
    w = (torch.randn(V, E, generator=g, device="cuda") * (2.5 / math.sqrt(E))).to(dtype)
    return x, w, torch.randint(0, V, (N,), generator=g, device="cuda")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("N,E,V", [
    (1, 8, 1), (1, 64, 15), (7, 72, 16), (128, 64, 127), (129, 128, 128), (3, 200, 129), (300, 256, 300),
    (1, 1024, 32003), (65, 1024, 5001), (257, 136, 20011), (700, 512, 2500), (5, 2048, 4097)])
def test_linear_logprobs(dtype, N, E, V):
    check_head(*operands(N + V, N, E, V, dtype))


@pytest.mark.parametrize("N,E,V", [(65, 520, 5001), (200, 1032, 3002), (3, 1544, 40), (300, 16384, 2500)])
def test_linear_logprobs_long_products(N, E, V):
    """Products of more columns than the tensor core sums at once (512): each of its 32 steps loses
    at most 2^-23 of the sum so far, on average no more than the logit, so logits shrink by at most
    2^-18 on average, and the entropy moves by that times their variance; 2^-18 more for a mean
    of what does not lean to one side."""
    from torchplusplus_b200 import ops
    x, w, t = operands(N + V, N, E, V, BF16)
    check_head(x, w, t)
    y = x.double() @ w.double().T
    p = torch.softmax(y, 1)
    var = (p * y * y).sum(1) - (p * y).sum(1) ** 2
    off = ops.linear_logprobs(x, w, t)[1].double() - oracle(y, t, 1.0, 0)[1]
    assert off.mean().abs() <= 2.0 ** -18 * (var.mean() + 1)


@pytest.mark.parametrize("temperature", [0.3, 2.0])
def test_linear_logprobs_temperature(temperature):
    check_head(*operands(1, 33, 256, 3001, BF16), temperature)


def test_linear_logprobs_peaked_and_growing():
    """Logits that grow along the vocabulary (every tile moves the reference), a sure token."""
    x, w, _ = operands(2, 40, 64, 4001, BF16)
    x[:, 0] = 4.0
    w[:, 0] = (torch.arange(4001, device="cuda") / 100).to(BF16)
    check_head(x, w, torch.full((40,), 4000, device="cuda"))
    check_head(x, w.flip(0).contiguous(), torch.arange(40, device="cuda"))


def test_linear_logprobs_strides_tokens_and_workspace():
    from torchplusplus_b200 import ops
    x, w, t = operands(3, 50, 128, 700, BF16)
    want = ops.linear_logprobs(x, w, t)
    xs = torch.empty(50, 136, dtype=BF16, device="cuda")
    xs[:, :128], xs[:, 128:] = x, math.nan
    ws = torch.empty(700, 144, dtype=BF16, device="cuda")
    ws[:, 16:], ws[:, :16] = w, math.nan
    room = torch.empty(ops.linear_logprobs_workspace_bytes(50, 700, 128), dtype=torch.uint8, device="cuda")
    for got in (ops.linear_logprobs(xs[:, :128], ws[:, 16:], t), ops.linear_logprobs(x, w, t, workspace=room),
                ops.linear_logprobs(x, w.T.contiguous().T, t)):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    t[3], t[4] = -5, 700
    lp, ent = ops.linear_logprobs(x, w, t)
    assert lp[3] == 0 and lp[4] == 0 and torch.equal(ent, want[1])
    x[9, 5] = math.nan
    lp, ent = ops.linear_logprobs(x, w, t)
    assert lp[9].isnan() and ent[9].isnan() and torch.equal(ent[10:], want[1][10:])


def test_scoring_of_a_prompt_agrees():
    """The head's scores and those of its written logits, as a scored prompt uses either."""
    from torchplusplus_b200 import ops
    x, w, t = operands(4, 100, 1024, 32003, BF16)
    lg = ops.linear(x, w)
    a, b = ops.linear_logprobs(x, w, t), ops.token_logprobs(lg, t)
    # the written logits are rounded to bf16
    d = 2.0 ** -8 * (x.double() @ w.double().T).abs().amax(1) * 1.01
    assert ((a[0] - b[0]).double().abs() <= 2 * d).all()


def test_refusals():
    from torchplusplus_b200 import ops
    x, t = logits(1, 4, 100, BF16), tokens_for(1, 4, 100)
    h, w, u = operands(1, 4, 64, 100, BF16)
    bad = [
        (ValueError, lambda: ops.token_logprobs(x[0], t)),
        (ValueError, lambda: ops.token_logprobs(x, t.int())),
        (ValueError, lambda: ops.token_logprobs(x, t[:3])),
        (ValueError, lambda: ops.token_logprobs(x, t, top=33)),
        (ValueError, lambda: ops.token_logprobs(x[:, :4], t, top=5)),
        (ValueError, lambda: ops.token_logprobs(x, t, top=-1)),
        (ValueError, lambda: ops.token_logprobs(x[:, :0], t)),
        (ValueError, lambda: ops.token_logprobs(x, t, temperature=0.0)),
        (ValueError, lambda: ops.token_logprobs(x, t, temperature=math.nan)),
        (ValueError, lambda: ops.token_logprobs(x, t, temperature=math.inf)),
        (TypeError, lambda: ops.token_logprobs(x.double(), t)),
        (RuntimeError, lambda: ops.token_logprobs(x, t.cpu())),
        (TypeError, lambda: ops.linear_logprobs(h.float(), w.float(), u)),
        (TypeError, lambda: ops.linear_logprobs(h, w.half(), u)),
        (ValueError, lambda: ops.linear_logprobs(h, w[:, :56], u)),
        (ValueError, lambda: ops.linear_logprobs(h[:, :60], w[:, :60], u)),
        (ValueError, lambda: ops.linear_logprobs(h, w[:0], u)),
        (ValueError, lambda: ops.linear_logprobs(h, w, u, temperature=-1.0)),
        (ops.N.TppError, lambda: ops.linear_logprobs(h, w, u, workspace=t)),
    ]
    for err, call in bad:
        with pytest.raises(err):
            call()
    assert ops.device_error() == 0
