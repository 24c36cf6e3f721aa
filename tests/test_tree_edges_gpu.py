"""Draft-tree operators where their plans, arguments and inputs leave the
ordinary: against the definitions in 64 bits of test_tree_gpu."""
import pytest
import torch

from .test_tree_gpu import (BF16, F16, UNIT, attention_oracle, contiguous_cache, make, pack,
                            paged_cache, verify_inputs)

pytestmark = pytest.mark.gpu


def attention(g, q, kc, vc, kt, vt, ctx, see, max_ctx=None, paged=False, mask=None, **kw):
    """attention_tree of CPU operands; max_ctx: the capacity given (the longest
    length unless set)."""
    from torchplusplus_b200 import ops
    lens = torch.tensor(ctx, dtype=torch.int32).cuda()
    mask = pack(see).cuda() if mask is None else mask.cuda()
    most = max(ctx) if max_ctx is None else max_ctx
    if paged:
        kp, vp, table = paged_cache(g, kc, vc)
        cols = max(1, (most + 63) // 64)
        wide = torch.full((len(ctx), cols), -1, dtype=torch.int32, device="cuda")
        wide[:, :table.shape[1]] = table
        return ops.attention_tree_paged(q.cuda(), kp, vp, wide, kt.cuda(), vt.cuda(), lens, most,
                                        mask, **kw)
    cap = max(most, 1)
    return ops.attention_tree(q.cuda(), contiguous_cache(kc, cap), contiguous_cache(vc, cap),
                              kt.cuda(), vt.cuda(), lens, most, mask, **kw)


def oracle(q, kc, vc, kt, vt, ctx, see, scale):
    """attention_oracle without a window, a head of a sequence at a time."""
    B, T, Hq, D = q.shape
    G, u = Hq // kt.shape[2], UNIT[q.dtype]
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b in range(B):
        n = int(ctx[b])
        hide = torch.zeros(T, n + T, dtype=torch.float64)
        hide[:, n:][~see[b]] = float("-inf")
        for h in range(Hq):
            k = torch.cat([kc[b][:, h // G], kt[b, :, h // G]]).double()
            v = torch.cat([vc[b][:, h // G], vt[b, :, h // G]]).double()
            x = q[b, :, h].double()
            w = torch.softmax(x @ k.T * scale + hide, 1)
            out[b, :, h] = o = w @ v
            a = w @ v.abs()
            big = (x.abs() @ k.abs().T * abs(scale) + hide).amax(1, keepdim=True)
            tol[b, :, h] = u * (a + o.abs()) + (2 * (D + 8) * 2.0 ** -24 * big + 2.0 ** -19) * a \
                + 2.0 ** -24
    return out, tol


# ------------------------------------------------------------------ the scale's sign
@pytest.mark.parametrize("scale", [-0.07, 0.0])
@pytest.mark.parametrize("B,T,Hq,Hkv,D,ctx", [
    (2, 5, 4, 2, 128, [100, 0]),          # 10 rows a unit
    (2, 40, 4, 2, 128, [100, 0]),         # 80 rows
    (1, 64, 16, 8, 64, [2500]),           # 128 rows, split
])
def test_attention_takes_any_scale(B, T, Hq, Hkv, D, ctx, scale):
    g = torch.Generator().manual_seed(31)
    q, kc, vc, kt, vt, see = make(g, B, T, Hq, Hkv, D, ctx, BF16)
    ref, tol = attention_oracle(q, kc, vc, kt, vt, ctx, see, -1, scale)
    o = attention(g, q, kc, vc, kt, vt, ctx, see, scale=scale).double().cpu()
    assert ((o - ref).abs() <= tol).all(), ((o - ref).abs() - tol).max()


# ------------------------------------------------------------------ the plans
# B, T, Hq, Hkv, D, ctx, capacity (None: the longest length)
PLANS = [
    (1, 64, 16, 8, 128, [3000], None),              # wide, each unit cut by itself
    (1, 64, 16, 8, 64, [2500], None),
    (2, 33, 2, 2, 128, [1900, 1500], None),         # 33 rows of 128
    (4, 40, 8, 2, 128, [3000, 10, 700, 0], None),   # wide, parts that straddle units
    (4, 40, 8, 2, 64, [3000, 10, 700, 0], None),
    (3, 20, 14, 2, 128, [40, 2900, 1111], None),    # 126 rows a unit, two row tiles
    (40, 40, 4, 2, 128, [2000 if b % 9 == 4 else 37 * b % 300 for b in range(40)], None),
    (70, 3, 4, 2, 128, [2500 if b % 23 == 7 else 41 * b % 350 for b in range(70)], None),
    (33, 16, 4, 2, 64, [0] * 32 + [3000], None),    # 32 rows, the last of two rounds
    (2, 5, 4, 2, 128, [200, 0], 4000),              # room for a cut that the lengths
    (2, 40, 4, 2, 128, [200, 700], 4000),           # turn out not to need
    (36, 4, 4, 2, 128, [9 * b for b in range(36)], 3000),
    (36, 40, 4, 2, 64, [9 * b for b in range(36)], 6000),
    (1, 8, 16, 8, 128, [2900], 30000),              # cut, far below the room
    (1, 50, 16, 8, 128, [2900], 30000),
]


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("case", PLANS, ids=lambda c: f"B{c[0]}T{c[1]}H{c[2]}/{c[3]}D{c[4]}"
                                                        f"n{max(c[5])}of{c[6]}")
def test_attention_of_every_plan(case, paged):
    B, T, Hq, Hkv, D, ctx, room = case
    dtype = F16 if paged else BF16
    g = torch.Generator().manual_seed(B * 1000 + T)
    q, kc, vc, kt, vt, see = make(g, B, T, Hq, Hkv, D, ctx, dtype)
    ref, tol = oracle(q, kc, vc, kt, vt, ctx, see, D ** -0.5)
    o = attention(g, q, kc, vc, kt, vt, ctx, see, room, paged).double().cpu()
    assert o.isfinite().all() and ((o - ref).abs() <= tol).all(), ((o - ref).abs() - tol).max()


@pytest.mark.parametrize("T,ctx,window", [(64, [3000], 2100), (40, [2000, 0, 900], 700),
                                          (8, [3000, 64], 1500)])
def test_attention_of_a_window_that_is_cut(T, ctx, window):
    g = torch.Generator().manual_seed(T)
    q, kc, vc, kt, vt, see = make(g, len(ctx), T, 4, 2, 128, ctx, BF16)
    ref, tol = attention_oracle(q, kc, vc, kt, vt, ctx, see, window, 128 ** -0.5)
    o = attention(g, q, kc, vc, kt, vt, ctx, see, window_left=window).double().cpu()
    assert ((o - ref).abs() <= tol).all(), ((o - ref).abs() - tol).max()


@pytest.mark.parametrize("B,T,Hq", [(1, 64, 4), (3, 40, 4), (1, 8, 4)])
def test_attention_nonfinite_values_of_a_unit_that_is_cut(B, T, Hq):
    """They reach the rows that see them and no others, whichever piece has them."""
    g = torch.Generator().manual_seed(41)
    ctx, D = [2900, 100, 1300][:B], 128
    q, kc, vc, kt, vt, see = make(g, B, T, Hq, 2, D, ctx, BF16)
    see[:, :, 2] = False
    see[:, 4, 2] = True
    ref, tol = attention_oracle(q, kc, vc, kt, vt, ctx, see, -1, D ** -0.5)
    vt[:, 2, :, 5] = float("inf")
    vt[:, 2, :, 70] = float("nan")
    o = attention(g, q, kc, vc, kt, vt, ctx, see).double().cpu()
    clean = torch.ones(B, T, Hq, D, dtype=torch.bool)
    clean[:, 4, :, 5] = clean[:, 4, :, 70] = False
    assert ((o - ref).abs() <= tol)[clean].all()
    assert (o[:, 4, :, 5] == float("inf")).all() and o[:, 4, :, 70].isnan().all()


# ------------------------------------------------------------------ verification
def test_verify_from_two_threads_with_different_vocabularies():
    """Each launch has the shared memory that its vocabulary takes, whatever the
    other thread's calls are."""
    import threading
    from torchplusplus_b200 import _native as N
    f = N.lib().tpp_verify_tree
    failed, keep = [], []

    def work(args, stream):
        for i in range(4000):
            if f(*args) != 0:
                failed.append(N.lib().tpp_last_error())
                return
            if i % 100 == 99:
                stream.synchronize()

    threads = []
    for V in (151936, 40000):
        lg = torch.zeros(1, 1, V, dtype=BF16, device="cuda")
        i64, i32 = (torch.zeros(2, dtype=t, device="cuda") for t in (torch.int64, torch.int32))
        path, count, nxt, u = i32.clone(), i32.clone(), i64.clone(), torch.zeros(1, device="cuda")
        stream = torch.cuda.Stream()
        keep.append((lg, i64, i32, path, count, nxt, u))
        args = (lg.data_ptr(), V, V, lg.data_ptr(), V, V, i64.data_ptr(), 1, i32.data_ptr(), 0,
                u.data_ptr(), 1, 1.0, path.data_ptr(), count.data_ptr(), nxt.data_ptr(), 1, 1, V,
                None, 0, N.dtype_code(BF16), stream.cuda_stream)
        threads.append(threading.Thread(target=work, args=(args, stream)))
    torch.cuda.synchronize()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed[0]


@pytest.mark.parametrize("T", [8, 64])
def test_attention_of_the_widest_window_over_many_keys(T):
    g = torch.Generator().manual_seed(61)
    ctx = [5000]
    q, kc, vc, kt, vt, see = make(g, 1, T, 16, 8, 128, ctx, BF16)
    call = lambda w: attention(g, q, kc, vc, kt, vt, ctx, see, window_left=w)
    full = call(-1)
    for w in (5000 + T, 2 ** 63 - 1):
        assert torch.equal(call(w), full)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("T,pads,V", [(2, 1, 501), (4, 3, 5003), (9, 20, 1001)])
def test_verify_nodes_without_a_token_change_nothing(draft, T, pads, V):
    """Trees filled up with nodes that hold no token (before and behind the real
    children, children of theirs among them) end as the trees without them: nothing
    was drawn for them, so they take nothing from the target's distribution."""
    from torchplusplus_b200 import ops
    g = torch.Generator().manual_seed(71 + T)
    B = 40
    logits, tokens, par, u, d = (x if x is None else x.cuda() for x in
                                 verify_inputs(g, B, T, V, BF16, False, draft))
    path, count, nxt = ops.verify_tree(logits, tokens, par, u, 1.0, d)
    # the first `lead` pads come right behind the root, the others last
    lead, N = pads // 2, T + pads
    at = torch.tensor([0] + list(range(1 + lead, T + lead)), device="cuda")    # of the real nodes
    big = [torch.randn(B, N, V, generator=g).to(BF16).cuda() for _ in range(2)]
    big[0][:, at] = logits
    if draft:
        big[1][:, at] = d
    tok2 = torch.full((B, N), -1, dtype=torch.int64, device="cuda")
    tok2[:, 1::2] = V + 3
    tok2[:, at] = tokens
    par2 = torch.zeros(B, N, dtype=torch.int32, device="cuda")
    par2[:, N - 1] = N - 2 if pads > 2 else 0
    par2[:, at] = torch.where(par >= 0, at[par.clamp_min(0).long()].int(), -1)
    u2 = torch.rand(B, N, generator=g).cuda()
    u2[:, at] = u
    path2, count2, nxt2 = ops.verify_tree(big[0], tok2, par2, u2, 1.0, big[1] if draft else None)
    assert torch.equal(count2, count) and torch.equal(nxt2, nxt)
    want = torch.where(path >= 0, at[path.clamp_min(0).long()].int(), -1)
    assert torch.equal(path2[:, :T], want) and (path2[:, T:] == -1).all()


def test_verify_emits_the_targets_distribution_from_padded_trees():
    """As the test of whole trees: chi-square with 9 degrees of freedom, 33.7 is
    passed once in 10^4."""
    from torchplusplus_b200 import ops
    g = torch.Generator().manual_seed(13)
    n, V = 60000, 10
    t = torch.randn(V, generator=g) * 1.2
    d = t + 0.8 * torch.randn(V, generator=g)
    want = torch.softmax(t.double(), 0) * n
    kid = torch.multinomial(torch.softmax(d, 0), n, True, generator=g)[:, None]
    tokens = torch.cat([torch.zeros_like(kid), kid, torch.full((n, 3), -1)], 1).cuda()
    par = torch.tensor([-1, 0, 0, 0, 0], dtype=torch.int32, device="cuda")
    lg, dl = (x.expand(1, 5, V).contiguous().cuda().expand(n, 5, V) for x in (t, d))
    path, count, nxt = ops.verify_tree(lg, tokens, par, torch.rand(n, 5, generator=g).cuda(), 1.0, dl)
    first = torch.where(count > 1, tokens.gather(1, path[:, 1:2].clamp_min(0).long())[:, 0], nxt)
    seen = torch.bincount(first.cpu(), minlength=V).double()
    assert float(((seen - want) ** 2 / want).sum()) < 33.7


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("T,chain", [(5, True), (12, False), (20, True)])
def test_verify_negative_uniforms_stand_for_zero(T, chain, draft):
    """For the tests of the children as for the draw: a token without weight is
    not accepted by them."""
    from torchplusplus_b200 import ops
    g = torch.Generator().manual_seed(81)
    logits, tokens, par, u, d = (x if x is None else x.cuda() for x in
                                 verify_inputs(g, 16, T, 777, BF16, chain, draft))
    none = torch.rand(16, T, generator=g) < 0.5       # their tokens have no weight
    none[0, 1:] = True
    for b, i in none[:, 1:].nonzero().tolist():
        logits[b, int(par[b, i + 1]), int(tokens[b, i + 1])] = float("-inf")
    low = torch.where(torch.rand(16, T, generator=g).cuda() < 0.5, u, -u)
    low[0], low[1] = -1.0, float("-inf")
    got = ops.verify_tree(logits, tokens, par, low, 1.0, d)
    assert int(got[1][0]) == 1
    for x, y in zip(got, ops.verify_tree(logits, tokens, par, low.clamp_min(0.0), 1.0, d)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("draft", [False, True])
def test_verify_uniforms_from_one_on_accept_the_only_token(draft):
    from torchplusplus_b200 import ops
    T = 4
    lg = torch.full((3, T, 300), float("-inf"), device="cuda")
    lg[:, :, 17] = 0.5
    u = torch.tensor([1.0, 3.0, float("inf")], device="cuda")[:, None].expand(3, T)
    path, count, nxt = ops.verify_tree(
        lg, torch.full((3, T), 17, device="cuda"),
        torch.arange(-1, T - 1, dtype=torch.int32, device="cuda"), u, 1.0, lg if draft else None)
    # with the draft's row equal to the target's, u * q < p holds for every u in [0, 1)
    assert count.tolist() == [T] * 3 and nxt.tolist() == [17] * 3


# ------------------------------------------------------------------ sliding windows
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("T,Hq,ctx,window", [(12, 4, [300, 2], 4), (12, 4, [50, 9], 0),
                                             (40, 4, [130, 0], 7), (70, 4, [500, 3], 65),
                                             (200, 2, [90, 1000], 100), (8, 4, [3000, 5], 1000)])
def test_attention_of_a_sliding_window_is_decodes(T, Hq, ctx, window, paged):
    """A chain's nodes see what decoding its tokens one after another with the
    same window sees: the keys [p - window, p], of the cache and of the tree."""
    from torchplusplus_b200 import ops
    from torchplusplus_b200.llmops import tree_mask
    g = torch.Generator().manual_seed(91)
    D = 128
    q, kc, vc, kt, vt, _ = make(g, 2, T, Hq, 2, D, ctx, BF16)
    par = torch.arange(-1, T - 1)
    o = attention(g, q, kc, vc, kt, vt, ctx, None, paged=paged, window_left=window,
                  mask=tree_mask(par, window)[0]).double().cpu()
    kall = [torch.cat([k, kt[b]]) for b, k in enumerate(kc)]
    vall = [torch.cat([v, vt[b]]) for b, v in enumerate(vc)]
    nobody = torch.zeros(2, 1, 1, dtype=torch.bool)
    cap = max(ctx) + T
    # (decode's caches are zero where nothing was written, as the framework makes them)
    kd, vd = contiguous_cache(kall, cap, 0.0), contiguous_cache(vall, cap, 0.0)
    for t in range(0, T, 1 if T < 50 else 9):
        # the oracle for the token at p = ctx + t: keys p - window to p, all its own cache
        lens = [n + t + 1 for n in ctx]
        low = [max(0, n + t - window) for n in ctx]
        part = [[x[b][low[b]:lens[b]] for b in range(2)] for x in (kall, vall)]
        ref, tol = attention_oracle(q[:, t:t + 1], *part, kt[:, :1], vt[:, :1],
                                    [len(x) for x in part[0]], nobody, -1, D ** -0.5)
        assert ((o[:, t:t + 1] - ref).abs() <= tol).all(), t
        d = ops.attention_decode(q[:, t].cuda(), kd, vd, torch.tensor(lens, dtype=torch.int32).cuda(),
                                 cap, window_left=window).double().cpu()
        assert ((d - o[:, t]).abs() <= 2 * tol[:, 0]).all(), t


def test_attention_of_a_sliding_window_over_a_branching_tree():
    from torchplusplus_b200.llmops import tree_mask
    g = torch.Generator().manual_seed(92)
    T, ctx, window, D = 48, [100, 3], 3, 128
    q, kc, vc, kt, vt, _ = make(g, 2, T, 4, 2, D, ctx, F16)
    par = torch.full((2, T), -1, dtype=torch.int32)
    for i in range(1, T):
        par[:, i] = (i * torch.rand(2, generator=g) ** 0.3).int()     # deep ones
    mask, depth = tree_mask(par, window)
    assert int(depth.max()) > 2 * window
    o = attention(g, q, kc, vc, kt, vt, ctx, None, window_left=window, mask=mask).double().cpu()
    for b in range(2):
        for t in range(T):
            path = [t]
            while par[b, path[-1]] >= 0:
                path.append(int(par[b, path[-1]]))
            path = path[::-1]                                         # the root first
            k, v = torch.cat([kc[b], kt[b, path]]), torch.cat([vc[b], vt[b, path]])
            k, v = k[-1 - window:], v[-1 - window:]
            ref, tol = attention_oracle(q[b:b + 1, t:t + 1], [k], [v], kt[:1, :1], vt[:1, :1],
                                        [len(k)], torch.zeros(1, 1, 1, dtype=torch.bool), -1, D ** -0.5)
            assert ((o[b, t] - ref[0, 0]).abs() <= tol[0, 0]).all(), (b, t)


# ------------------------------------------------------------------ q/k norm + RoPE
@pytest.mark.parametrize("B,T", [(1, 3), (64, 64)])
def test_qk_norm_rope_positions_outside_the_table_are_zero_without_an_eps(B, T):
    from torchplusplus_b200 import ops
    D = 128
    g = torch.Generator().manual_seed(101)
    qkv = torch.randn(B, T, 8 * D, generator=g).to(BF16).cuda()
    w = torch.ones(D, dtype=BF16, device="cuda")
    cos = torch.ones(10, D, device="cuda")
    pos = torch.randint(0, 10, (B, T), generator=g).int()
    pos[0, 1], pos[-1, -1] = -1, 10
    q, k = ops.qk_norm_rope_tree(qkv, w, w, 0.0, cos, cos, pos.cuda(), 4, 2)
    out = (pos < 0) | (pos >= 10)
    for x in (q, k):
        assert (x.cpu()[out] == 0).all() and x.isfinite().all()
