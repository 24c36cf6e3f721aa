"""Draft-tree operators against their definitions in 64 bits: attention over
cache and tree, q/k norm and rotary positions, verification, commit."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
# unit roundoff (half an ulp over the value) of the storage types
UNIT = {F16: 2.0 ** -11, BF16: 2.0 ** -8}


def random_parents(g, B, T):
    par = torch.full((B, T), -1, dtype=torch.int32)
    for i in range(1, T):
        par[:, i] = (torch.rand(B, generator=g) * i).int()
    return par


def ancestors(par):
    B, T = par.shape
    see = torch.zeros(B, T, T, dtype=torch.bool)
    for b in range(B):
        for i in range(T):
            if i:
                see[b, i] = see[b, par[b, i]]
            see[b, i, i] = True
    return see


def pack(see):
    B, T, _ = see.shape
    out = torch.zeros(B, T, (T + 63) // 64, dtype=torch.int64)
    for j in range(T):
        out[:, :, j // 64] |= see[:, :, j].long() << (j % 64)
    return out


def attention_oracle(q, kc, vc, kt, vt, ctx, see, window, scale):
    """o and its error bound, both [B,T,Hq,D] in 64 bits.  kc/vc: a list of
    [ctx_b, Hkv, D].  The bound: the probabilities and the result are each
    rounded once to the storage type (u * sum w|v| + u|o|), and the scores carry
    the error of an fp32 dot product of D terms, which turns into a relative
    error of every weight (twice: in the sum and in the norm)."""
    B, T, Hq, D = q.shape
    Hkv = kt.shape[2]
    u = UNIT[q.dtype]
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b in range(B):
        n = int(ctx[b])
        vis = torch.cat([torch.ones(T, n, dtype=torch.bool), see[b]], 1)
        if window >= 0:
            low = n + see[b].sum(1) - 1 - window
            vis[:, :n] &= torch.arange(n)[None] >= low[:, None]
        for h in range(Hq):
            kv = h // (Hq // Hkv)
            k = torch.cat([kc[b][:, kv], kt[b, :, kv]]).double()
            v = torch.cat([vc[b][:, kv], vt[b, :, kv]]).double()
            for t in range(T):
                at = vis[t].nonzero()[:, 0]
                if not len(at):
                    continue
                x = q[b, t, h].double()
                s = (k[at] @ x) * scale
                w = torch.softmax(s, 0)
                o = w @ v[at]
                a = w @ v[at].abs()
                big = ((k[at].abs() @ x.abs()) * abs(scale)).max()
                out[b, t, h] = o
                tol[b, t, h] = u * (a + o.abs()) + (2 * (D + 8) * 2.0 ** -24 * big + 2.0 ** -19) * a \
                    + 2.0 ** -24  # fp16 results under 2^-14 round to multiples of 2^-24
    return out, tol


def make(g, B, T, Hq, Hkv, D, ctx, dtype, spread=2.0):
    q = (spread * torch.randn(B, T, Hq, D, generator=g)).to(dtype)
    kt = torch.randn(B, T, Hkv, D, generator=g).to(dtype)
    vt = torch.randn(B, T, Hkv, D, generator=g).to(dtype)
    kc = [torch.randn(n, Hkv, D, generator=g).to(dtype) for n in ctx]
    vc = [torch.randn(n, Hkv, D, generator=g).to(dtype) for n in ctx]
    see = ancestors(random_parents(g, B, T))
    return q, kc, vc, kt, vt, see


def contiguous_cache(rows, cap, fill=float("nan")):
    """[B,Hkv,cap,D]; what no sequence has written is `fill`."""
    Hkv, D = rows[0].shape[1:]
    c = torch.full((len(rows), Hkv, cap, D), fill, dtype=rows[0].dtype)
    for b, r in enumerate(rows):
        c[b, :, :len(r)] = r.transpose(0, 1)
    return c.cuda()


def paged_cache(g, k, v, fill=float("nan")):
    """Pools of shuffled blocks and the table; unwritten rows are `fill`."""
    B, (Hkv, D) = len(k), k[0].shape[1:]
    nb = max(1, max((len(r) + 63) // 64 for r in k))
    table = torch.randperm(B * nb + 3, generator=g)[:B * nb].view(B, nb).int()
    pools = []
    for x in (k, v):
        pool = torch.full((B * nb + 3, Hkv, 64, D), fill, dtype=k[0].dtype)
        for b, r in enumerate(x):
            for i in range(0, len(r), 64):
                part = r[i:i + 64].transpose(0, 1)
                pool[table[b, i // 64], :, :part.shape[1]] = part
        pools.append(pool.cuda())
    return pools[0], pools[1], table.cuda()


def run_tree(g, q, kc, vc, kt, vt, ctx, see, window=-1, paged=False, **kw):
    from torchplusplus_b200 import ops
    lens = torch.tensor(ctx, dtype=torch.int32).cuda()
    mask = pack(see).cuda()
    if paged:
        kp, vp, table = paged_cache(g, kc, vc)
        return ops.attention_tree_paged(q.cuda(), kp, vp, table, kt.cuda(), vt.cuda(), lens,
                                        max(ctx), mask, window_left=window, **kw)
    cap = max(max(ctx), 1) + 70
    return ops.attention_tree(q.cuda(), contiguous_cache(kc, cap), contiguous_cache(vc, cap),
                              kt.cuda(), vt.cuda(), lens, max(ctx), mask, window_left=window,
                              **kw)


CASES = [
    # B, T, Hq, Hkv, D, ctx, window
    (1, 1, 2, 2, 64, [0], -1),                     # one node, nothing before it
    (1, 1, 16, 8, 128, [1], -1),
    (2, 5, 16, 8, 128, [130, 63], -1),
    (3, 8, 4, 2, 128, [64, 65, 0], -1),            # 16 rows, ends on and past a tile
    (2, 13, 8, 2, 128, [127, 300], -1),            # 52 rows
    (2, 17, 2, 2, 64, [200, 1], -1),               # 17 rows: the second row group has one
    (1, 33, 4, 4, 64, [129], -1),
    (1, 64, 4, 2, 128, [511], -1),                 # 128 rows
    (2, 65, 2, 1, 128, [70, 192], -1),             # the mask's second word
    (1, 130, 3, 1, 64, [100], -1),
    (1, 256, 2, 2, 128, [33], -1),
    (2, 9, 14, 2, 128, [90, 400], -1),             # 7 query heads a kv head
    (1, 4, 32, 1, 64, [77], -1),                   # one kv head
    (2, 12, 4, 2, 128, [300, 40], 100),            # a window whose edge differs by depth
    (2, 40, 4, 2, 64, [500, 129], 64),
    (1, 6, 4, 2, 128, [200], 0),                   # a window of the position alone
    (1, 20, 4, 2, 128, [200], 3),                  # a window shorter than the tree is deep
    (5, 3, 4, 2, 128, [2100, 0, 17, 640, 1999], -1),   # ragged, long enough to be split
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"B{c[0]}T{c[1]}H{c[2]}/{c[3]}D{c[4]}w{c[6]}")
def test_attention(case, paged, dtype):
    B, T, Hq, Hkv, D, ctx, window = case
    g = torch.Generator().manual_seed(100 + T)
    q, kc, vc, kt, vt, see = make(g, B, T, Hq, Hkv, D, ctx, dtype)
    o = run_tree(g, q, kc, vc, kt, vt, ctx, see, window, paged)
    ref, tol = attention_oracle(q, kc, vc, kt, vt, ctx, see, window, 1 / math.sqrt(D))
    err = (o.double().cpu() - ref).abs()
    assert o.isfinite().all() and (err <= tol).all(), ((err - tol).max(), err.max())


@pytest.mark.parametrize("T,Hq", [(7, 2), (40, 4), (70, 4)])
def test_attention_rows_that_see_nothing_are_zero(T, Hq):
    g = torch.Generator().manual_seed(3)
    q, kc, vc, kt, vt, see = make(g, 2, T, Hq, 2, 128, [0, 90], BF16)
    see[0, T // 2] = False          # no context, no nodes
    see[0, :, T - 1] = False        # a node that nobody sees, itself included
    see[1, 3] = False               # context only
    o = run_tree(g, q, kc, vc, kt, vt, [0, 90], see).double().cpu()
    ref, tol = attention_oracle(q, kc, vc, kt, vt, [0, 90], see, -1, 128 ** -0.5)
    assert (o[0, T // 2] == 0).all()
    assert ((o - ref).abs() <= tol).all()


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("T,Hq,ctx", [(6, 2, 100), (30, 4, 100), (64, 4, 300), (9, 4, 1500)])
def test_attention_masked_nonfinite_values_have_no_effect(T, Hq, ctx, paged):
    """A node's K/V reach only the rows that see it, whatever they hold (rows
    past the context are NaN in every test here)."""
    g = torch.Generator().manual_seed(4)
    q, kc, vc, kt, vt, see = make(g, 1, T, Hq, 2, 128, [ctx], BF16)
    ref, tol = attention_oracle(q, kc, vc, kt, vt, [ctx], see, -1, 128 ** -0.5)
    see[0, :, 2] = False            # nobody sees node 2
    see[0, 4, 2] = True             # but node 4
    base, btol = attention_oracle(q, kc, vc, kt, vt, [ctx], see, -1, 128 ** -0.5)
    kt2, vt2 = kt.clone(), vt.clone()
    kt2[0, 2] = float("nan")
    vt2[0, 2] = float("nan")
    o = run_tree(g, q, kc, vc, kt2, vt2, [ctx], see, paged=paged).double().cpu()
    rest = torch.arange(T) != 4
    assert ((o - base).abs() <= btol)[:, rest].all()
    assert o[0, 4].isnan().all()
    vt3 = vt.clone()                # infinities in some dims of a value
    vt3[0, 2, :, 5] = float("inf")
    vt3[0, 2, :, 70] = -float("inf")
    o = run_tree(g, q, kc, vc, kt, vt3, [ctx], see, paged=paged).double().cpu()
    assert ((o - base).abs() <= btol)[:, rest].all()
    assert (o[0, 4, :, 5] == float("inf")).all() and (o[0, 4, :, 70] == -float("inf")).all()
    dims = torch.ones(128, dtype=torch.bool)
    dims[5] = dims[70] = False
    assert ((o - base).abs() <= btol)[0, 4][:, dims].all()


def test_attention_nonfinite_below_a_window():
    """Cache rows that a window hides from a node, or from all."""
    g = torch.Generator().manual_seed(5)
    T, ctx, w = 10, 400, 150
    q, kc, vc, kt, vt, see = make(g, 1, T, 4, 2, 128, [ctx], F16)
    see = torch.tril(torch.ones(T, T, dtype=torch.bool))[None]     # a chain
    base, tol = attention_oracle(q, kc, vc, kt, vt, [ctx], see, w, 128 ** -0.5)
    for x in (kc[0], vc[0]):
        x[:ctx + 4 - w] = float("nan")       # rows that nodes 4.. do not see
    o = run_tree(g, q, kc, vc, kt, vt, [ctx], see, w).double().cpu()
    assert ((o - base).abs() <= tol)[0, 4:].all()
    assert o[0, :4].isnan().all()


def test_attention_strided_operands_and_output():
    from torchplusplus_b200 import ops
    g = torch.Generator().manual_seed(6)
    B, T, Hq, Hkv, D, ctx = 2, 11, 4, 2, 128, [150, 77]
    q, kc, vc, kt, vt, see = make(g, B, T, Hq, Hkv, D, ctx, BF16)
    ref, tol = attention_oracle(q, kc, vc, kt, vt, ctx, see, -1, 0.05)
    qh = q.cuda().permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)      # heads outside
    kv = torch.cat([kt.flatten(2), vt.flatten(2)], 2).cuda()                # one row a node
    ktv = kv[..., :Hkv * D].view(B, T, Hkv, D)
    vtv = kv[..., Hkv * D:].view(B, T, Hkv, D)
    cache = torch.full((B, 2, Hkv, 400, D), float("nan"), dtype=BF16, device="cuda")
    cache[:, 0, :, :350] = contiguous_cache(kc, 350)
    cache[:, 1, :, :350] = contiguous_cache(vc, 350)
    out = torch.full((B, Hq, T, D + 2), 7.0, dtype=BF16, device="cuda")
    view = out.permute(0, 2, 1, 3)[..., :D]
    mask = pack(see).cuda()
    lens = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    ops.attention_tree(qh, cache[:, 0], cache[:, 1], ktv, vtv, lens, 200, mask, scale=0.05,
                       out=view)
    assert ((view.double().cpu() - ref).abs() <= tol).all()
    assert (out[..., D:] == 7).all()
    # operands whose rows start off 16 bytes are copied
    odd = torch.empty(B * T * Hq * D + 1, dtype=BF16, device="cuda")[1:].view(B, T, Hq, D)
    odd.copy_(q)
    o2 = ops.attention_tree(odd, cache[:, 0], cache[:, 1], ktv, vtv, lens, 200, mask, scale=0.05)
    assert torch.equal(o2, view)


def test_attention_shared_mask_lengths_out_of_range_and_missing_blocks():
    from torchplusplus_b200 import ops
    g = torch.Generator().manual_seed(7)
    B, T, ctx = 3, 6, [100, 100, 0]
    q, kc, vc, kt, vt, see = make(g, B, T, 4, 2, 128, ctx, F16)
    see = see[:1].expand(B, T, T).contiguous()
    ref, tol = attention_oracle(q, kc, vc, kt, vt, ctx, see, -1, 128 ** -0.5)
    k, v = contiguous_cache(kc, 130), contiguous_cache(vc, 130)
    lens = torch.tensor([100, 5000, -3], dtype=torch.int32, device="cuda")  # clamped to [0, 100]
    o = ops.attention_tree(q.cuda(), k, v, kt.cuda(), vt.cuda(), lens, 100, pack(see)[0].cuda())
    assert ((o.double().cpu() - ref).abs() <= tol).all()
    # a block number outside the pool stands for 64 keys of zeros
    kp, vp, table = paged_cache(g, kc, vc, 0.0)
    table[0, 0], table[1, 0] = -1, 10 ** 6
    for b in (0, 1):
        kc[b][:64] = 0
        vc[b][:64] = 0
    ref, tol = attention_oracle(q, kc, vc, kt, vt, ctx, see, -1, 128 ** -0.5)
    o = ops.attention_tree_paged(q.cuda(), kp, vp, table, kt.cuda(), vt.cuda(), lens, 100,
                                 pack(see)[0].cuda())
    assert ((o.double().cpu() - ref).abs() <= tol).all()


@pytest.mark.parametrize("T", [3, 40])
def test_attention_empty_cache_wide_windows_and_shared_operands(T):
    from torchplusplus_b200 import ops
    g = torch.Generator().manual_seed(17)
    B, D = 2, 128
    q, kc, vc, kt, vt, see = make(g, B, T, 4, 2, D, [100, 60], BF16)
    # a cache without rows
    none = [x[:0] for x in kc]
    ref, tol = attention_oracle(q, none, none, kt, vt, [0, 0], see, -1, D ** -0.5)
    e = torch.zeros(B, 2, 0, D, dtype=BF16, device="cuda")
    z = torch.zeros(B, dtype=torch.int32, device="cuda")
    o = ops.attention_tree(q.cuda(), e, e, kt.cuda(), vt.cuda(), z, 0, pack(see).cuda())
    assert ((o.double().cpu() - ref).abs() <= tol).all()
    # windows that reach past every row
    k, v = contiguous_cache(kc, 100), contiguous_cache(vc, 100)
    lens = torch.tensor([100, 60], dtype=torch.int32, device="cuda")
    call = lambda **kw: ops.attention_tree(q.cuda(), k, v, kt.cuda(), vt.cuda(), lens, 100,
                                           pack(see).cuda(), **kw)
    full = call()
    for w in (100 + T, 2 ** 31, 2 ** 63 - 1):
        assert torch.equal(call(window_left=w), full)
    # every sequence the same tree: q, k and v expanded over the batch
    one = [x[:1].cuda() for x in (q, kt, vt)]
    a = ops.attention_tree(one[0].expand(B, T, 4, D), k, v, one[1].expand(B, T, 2, D),
                           one[2].expand(B, T, 2, D), lens, 100, pack(see)[0].cuda())
    b = ops.attention_tree(*(x.repeat(B, 1, 1, 1) if i in (0, 3, 4) else x for i, x in
                             enumerate((one[0], k, v, one[1], one[2]))), lens, 100,
                           pack(see)[:1].repeat(B, 1, 1).cuda())
    assert torch.equal(a, b)


@pytest.mark.parametrize("T", [4, 40])
def test_attention_offsets_past_32_bits(T):
    """A cache of more than 2^31 elements a sequence, read at its end."""
    from torchplusplus_b200 import ops
    g = torch.Generator().manual_seed(8)
    D, cap, w = 128, (1 << 24) + 200, 150
    kc = torch.empty(2, 1, cap, D, dtype=F16, device="cuda")
    vc = torch.empty(2, 1, cap, D, dtype=F16, device="cuda")
    ctx = cap - 3
    q, k, v, kt, vt, see = make(g, 2, T, 2, 1, D, [200, 200], F16)
    for b in range(2):
        kc[b, 0, ctx - 200:ctx] = k[b][:, 0].cuda()
        vc[b, 0, ctx - 200:ctx] = v[b][:, 0].cuda()
    lens = torch.full((2,), ctx, dtype=torch.int32, device="cuda")
    o = ops.attention_tree(q.cuda(), kc, vc, kt.cuda(), vt.cuda(), lens, ctx, pack(see).cuda(),
                           window_left=w)
    ref, tol = attention_oracle(q, k, v, kt, vt, [200, 200], see, w, D ** -0.5)
    assert ((o.double().cpu() - ref).abs() <= tol).all()


def test_attention_is_the_same_on_another_stream_and_every_time():
    from torchplusplus_b200 import ops
    g = torch.Generator().manual_seed(9)
    ctx = [3000, 1200]
    q, kc, vc, kt, vt, see = make(g, 2, 24, 16, 8, 128, ctx, BF16)
    a = [x.cuda() for x in (q, kt, vt)]
    k, v = contiguous_cache(kc, 3000), contiguous_cache(vc, 3000)
    lens = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    mask = pack(see).cuda()
    call = lambda: ops.attention_tree(a[0], k, v, a[1], a[2], lens, 3000, mask)
    first = call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        outs = [call() for _ in range(20)]
    side.synchronize()
    assert all(torch.equal(first, o) for o in outs)


def test_attention_refusals():
    from torchplusplus_b200 import ops
    from torchplusplus_b200 import TppError
    z = lambda *s, dt=BF16: torch.zeros(*s, dtype=dt, device="cuda")
    lens = z(1, dt=torch.int32)
    mask = z(4, 1, dt=torch.int64)
    q, k, t = z(1, 4, 4, 128), z(1, 2, 64, 128), z(1, 4, 2, 128)
    good = dict(q=q, k_cache=k, v_cache=k, k_tree=t, v_tree=t, ctx_lens=lens, max_ctx=64, mask=mask)
    ops.attention_tree(**good)
    bad = [
        (dict(q=q.cpu()), RuntimeError), (dict(q=q.float()), TypeError),
        (dict(k_cache=k.half()), TypeError), (dict(max_ctx=65), ValueError),
        (dict(max_ctx=-1), ValueError), (dict(q=z(1, 4, 3, 128)), ValueError),
        (dict(k_tree=z(1, 3, 2, 128)), ValueError), (dict(mask=mask.int()), ValueError),
        (dict(mask=z(4, 2, dt=torch.int64)), ValueError), (dict(ctx_lens=lens.long()), ValueError),
        (dict(v_cache=z(1, 2, 80, 128)), ValueError), (dict(q=z(4, 4, 128)), ValueError),
        (dict(out=z(1, 4, 4, 64)), ValueError),
        (dict(q=z(1, 300, 4, 128), k_tree=z(1, 300, 2, 128), v_tree=z(1, 300, 2, 128),
              mask=z(300, 5, dt=torch.int64)), TppError),
        (dict(q=z(1, 4, 4, 96), k_cache=z(1, 2, 64, 96), v_cache=z(1, 2, 64, 96),
              k_tree=z(1, 4, 2, 96), v_tree=z(1, 4, 2, 96)), TppError),
    ]
    for change, err in bad:
        with pytest.raises(err):
            ops.attention_tree(**{**good, **change})
    p = z(3, 2, 64, 128)
    tbl = z(1, 1, dt=torch.int32)
    pg = dict(q=q, k_pool=p, v_pool=p, block_table=tbl, k_tree=t, v_tree=t, ctx_lens=lens,
              max_ctx=64, mask=mask)
    ops.attention_tree_paged(**pg)
    for change in (dict(max_ctx=65), dict(k_pool=z(3, 2, 32, 128)), dict(block_table=tbl.long())):
        with pytest.raises(ValueError):
            ops.attention_tree_paged(**{**pg, **change})
    assert ops.attention_tree(**{**good, **dict(q=q[:0], k_cache=k[:0], v_cache=k[:0],
                                                k_tree=t[:0], v_tree=t[:0],
                                                ctx_lens=lens[:0])}).shape[0] == 0


# ------------------------------------------------------------------ q/k norm + RoPE
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tdtype", [F16, torch.float32])
@pytest.mark.parametrize("B,T,Hq,Hkv,D", [(1, 1, 1, 1, 16), (2, 7, 4, 2, 64), (3, 5, 16, 8, 128),
                                          (1, 33, 3, 1, 256), (2, 2, 5, 5, 32)])
@pytest.mark.parametrize("norm", [True, False])
def test_qk_norm_rope(B, T, Hq, Hkv, D, norm, dtype, tdtype):
    from torchplusplus_b200 import ops
    g = torch.Generator().manual_seed(D)
    W, rows = (Hq + 2 * Hkv) * D, 50
    qkv = torch.randn(B, T, W + 8, generator=g).to(dtype)
    wq = (1 + 0.2 * torch.randn(D, generator=g)).to(dtype) if norm else None
    wk = (1 + 0.2 * torch.randn(D, generator=g)).to(dtype) if norm else None
    ang = torch.rand(rows, D // 2, generator=g) * 6
    ang = torch.cat([ang, ang], 1)
    cos, sin = ang.cos().to(tdtype), ang.sin().to(tdtype)
    pos = torch.randint(0, rows, (B, T), generator=g).int()
    cu = lambda t: None if t is None else t.cuda()
    qkv_v = qkv.cuda()[..., :W]                        # a row stride of its own
    q, k = ops.qk_norm_rope_tree(qkv_v, cu(wq), cu(wk), 1e-6, cos.cuda(), sin.cuda(), pos.cuda(),
                                 Hq, Hkv)
    x = qkv[..., :W].double().view(B, T, Hq + 2 * Hkv, D)
    for got, part, w in ((q, x[:, :, :Hq], wq), (k, x[:, :, Hq:Hq + Hkv], wk)):
        if w is not None:
            part = part / (part.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        c, s = (t.double()[pos.long()][:, :, None] for t in (cos, sin))
        half = torch.cat([-part[..., D // 2:], part[..., :D // 2]], -1)
        ref = part * c + half * s
        # one rounding to the type, and an fp32 evaluation of a dozen roundings
        tol = UNIT[dtype] * ref.abs() + 16 * 2.0 ** -24 * ((part * c).abs() + (half * s).abs()) + 2.0 ** -24
        assert ((got.double().cpu() - ref).abs() <= tol).all()


def test_qk_norm_rope_positions_outside_the_table_and_refusals():
    from torchplusplus_b200 import ops
    qkv = torch.randn(1, 4, 4 * 64, device="cuda").half()
    cos = torch.ones(10, 64, device="cuda").half()
    pos = torch.tensor([[0, -1, 10, 9]], dtype=torch.int32, device="cuda")
    q, k = ops.qk_norm_rope_tree(qkv, None, None, 1e-6, cos, cos, pos, 2, 1)
    assert (q[0, 1:3] == 0).all() and (k[0, 1:3] == 0).all()
    assert (q[0, 0] != 0).any() and (q[0, 3] != 0).any()
    for args, err in (((qkv.cpu(), None, None, 1e-6, cos, cos, pos, 2, 1), RuntimeError),
                      ((qkv, None, None, 1e-6, cos, cos, pos.long(), 2, 1), ValueError),
                      ((qkv, None, None, 1e-6, cos, cos, pos[:, :3], 2, 1), ValueError),
                      ((qkv, None, None, 1e-6, cos, cos, pos, 3, 1), ValueError),
                      ((qkv.float(), None, None, 1e-6, cos, cos, pos, 2, 1), TypeError),
                      ((qkv, cos[0, :32], None, 1e-6, cos, cos, pos, 2, 1), ValueError)):
        with pytest.raises(err):
            ops.qk_norm_rope_tree(*args)


# ------------------------------------------------------------------ verification
def verify_oracle(logits, tokens, par, u, temp, draft):
    """One sequence's walk in 64 bits: (path, next, the smallest distance of a
    decision from flipping, relative to the mass it was made over)."""
    T, V = logits.shape

    def weights(row):
        x = torch.where(row.isnan(), -math.inf, row.double())
        m = x.max()
        if not m.isfinite():
            return torch.zeros(V, dtype=torch.float64)
        return ((x - m) / temp).exp()

    path, cur, margin = [0], 0, 1.0
    while True:
        if temp == 0:
            x = torch.where(logits[cur].isnan(), -math.inf, logits[cur].double())
            top = int((x == x.max()).nonzero()[0, 0]) if x.max() > -math.inf else -1
            p = torch.zeros(V, dtype=torch.float64)
            if top >= 0:
                p[top] = 1
        else:
            p = weights(logits[cur])
            p = p / p.sum() if p.sum() > 0 else p
        kids = [i for i in range(cur + 1, T) if par[i] == cur]
        q = None
        if draft is not None and temp > 0 and kids:
            q = weights(draft[cur])
            q = q / q.sum() if q.sum() > 0 else q
        took = None
        for i in kids:
            t = int(tokens[i])
            pt = float(p[t]) if 0 <= t < V else 0.0
            if temp == 0:
                ok = pt > 0
            elif q is None:
                left = float(p.sum())
                ok = float(u[i]) * left < pt
                margin = min(margin, abs(float(u[i]) * left - pt))
                if not ok and 0 <= t < V:
                    p[t] = 0
            else:
                qt = float(q[t]) if 0 <= t < V else 0.0
                ok = 0 <= t < V and float(u[i]) * qt < pt
                margin = min(margin, abs(float(u[i]) * qt - pt) / max(qt, pt, 1e-300))
                if not ok:
                    r = (p - q).clamp_min(0)
                    if 0 < r.sum() < 1e-6:      # a residual of rounding errors
                        margin = 0
                    p = r / r.sum() if r.sum() > 0 else p
            if ok:
                took = i
                break
        if took is None:
            break
        path.append(took)
        cur = took
    if p.sum() <= 0:
        return path, -1, margin
    if temp == 0:
        return path, int(p.argmax()), 1.0
    cum = p.cumsum(0)
    at = float(u[0]) * float(cum[-1])
    nxt = int((cum <= at).sum())
    margin = min(margin, float((cum - at).abs().min()) / float(cum[-1]))
    return path, nxt, margin


def check_verify(logits, tokens, par, u, temp, draft, least=0.8):
    from torchplusplus_b200 import ops
    B, T, V = logits.shape
    path, count, nxt = ops.verify_tree(logits.cuda(), tokens.cuda(), par.cuda(),
                                       None if u is None else u.cuda(), temp,
                                       None if draft is None else draft.cuda())
    path, count, nxt = path.cpu(), count.cpu(), nxt.cpu()
    sure = 0
    for b in range(B):
        pb = par if par.dim() == 1 else par[b]
        ref, tok, margin = verify_oracle(logits[b], tokens[b], pb, None if u is None else u[b],
                                         temp, None if draft is None else draft[b])
        # fp32 weights are within 2^-21 or so of the exact ones
        if temp > 0 and margin < 4e-6:
            continue
        sure += 1
        assert path[b].tolist() == ref + [-1] * (T - len(ref)), (b, ref, path[b])
        assert int(count[b]) == len(ref) and int(nxt[b]) == tok, (b, tok, int(nxt[b]))
    assert sure >= least * B
    return path, count, nxt


def verify_inputs(g, B, T, V, dtype, chain, draft, spread=2.0):
    logits = (spread * torch.randn(B, T, V, generator=g)).to(dtype)
    par = torch.arange(-1, T - 1).int().expand(B, T).contiguous() if chain else random_parents(g, B, T)
    d = (logits.float() + 0.7 * torch.randn(B, T, V, generator=g)).to(dtype) if draft else None
    tokens = torch.zeros(B, T, dtype=torch.int64)
    for b in range(B):
        for i in range(1, T):
            x = (d if draft else logits)[b, par[b, i]].float()
            # the likelier tokens, some of them twice among siblings
            tokens[b, i] = x.topk(min(4, V)).indices[int(torch.randint(0, min(4, V), (1,), generator=g))]
    u = torch.rand(B, T, generator=g)
    return logits, tokens, par, u, d


@pytest.mark.parametrize("dtype", [BF16, F16, torch.float32])
@pytest.mark.parametrize("temp", [0.0, 0.7, 1.0])
@pytest.mark.parametrize("B,T,V,chain,draft", [
    (3, 1, 17, True, False),          # the root alone: a draw
    (16, 5, 1000, True, True),
    (16, 9, 32003, True, True),       # rows that start off 16 bytes
    (16, 12, 257, False, False),
    (16, 40, 4099, False, False),
    (16, 12, 501, False, True),       # several draws from one draft distribution
    (2, 5, 151936, True, True),
    (4, 64, 7, False, False),
    (3, 4, 1, True, False),           # one token only
])
def test_verify(B, T, V, chain, draft, temp, dtype):
    g = torch.Generator().manual_seed(T * 1000 + V)
    check_verify(*verify_inputs(g, B, T, V, dtype, chain, draft)[:4], temp,
                 verify_inputs(torch.Generator().manual_seed(T * 1000 + V), B, T, V, dtype, chain,
                               draft)[4], least=0.5 if V > 1000 else 0.8)


def test_verify_greedy_takes_the_lowest_of_equal_logits():
    g = torch.Generator().manual_seed(1)
    logits = torch.randint(-3, 4, (8, 6, 3001), generator=g).to(BF16)   # many ties
    tokens = torch.zeros(8, 6, dtype=torch.int64)
    for i in range(1, 6):
        tokens[:, i] = logits[:, i - 1].float().argmax(-1)
        for b in range(8):
            tokens[b, i] = (logits[b, i - 1] == logits[b, i - 1].max()).nonzero()[0, 0]
    path, count, _ = check_verify(logits, tokens, torch.arange(-1, 5).int(), None, 0.0, None)
    assert (count == 6).all()


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("temp", [0.0, 1.0])
def test_verify_nan_infinite_and_empty_rows(draft, temp):
    g = torch.Generator().manual_seed(2)
    logits, tokens, par, u, d = verify_inputs(g, 6, 5, 777, torch.float32, True, draft)
    logits[0, 0] = -math.inf                         # no weight at the root
    logits[1, 0, ::2] = math.nan                     # NaN counts as -inf
    logits[2, 0, 5:] = -math.inf
    logits[3, 0] = math.nan
    logits[4, 0, 100:] = torch.finfo(torch.float32).min
    tokens[5, 1:] = torch.tensor([-1, 777, 5, 6])    # tokens that are none
    if draft:
        d[2, 0, :3] = -math.inf
        d[5, 0] = -math.inf
    _, count, nxt = check_verify(logits, tokens, par, u, temp, d, least=0.6)
    assert int(nxt[0]) == -1 and int(nxt[3]) == -1 and int(count[0]) == 1 and int(count[5]) == 1
    assert int(nxt[1]) % 2 == 1 or int(count[1]) > 1


def test_verify_emits_the_targets_distribution():
    """First emitted token over many draws: chi-square against the target's
    softmax (9 degrees of freedom: 33.7 is passed once in 10^4)."""
    from torchplusplus_b200 import ops
    g = torch.Generator().manual_seed(11)
    n, V = 60000, 10
    t = torch.randn(V, generator=g) * 1.2
    d = t + 0.8 * torch.randn(V, generator=g)
    want = torch.softmax(t.double(), 0) * n
    par = torch.tensor([-1, 0, 0], dtype=torch.int32)
    for with_draft in (True, False):
        if with_draft:   # both children drawn from the draft
            kids = torch.multinomial(torch.softmax(d, 0), n * 2, True, generator=g).view(n, 2)
        else:            # any two proposals
            kids = torch.tensor([[3, 7]]).expand(n, 2)
        tokens = torch.cat([torch.zeros(n, 1, dtype=torch.int64), kids], 1).cuda()
        u = torch.rand(n, 3, generator=g).cuda()
        lg = t.expand(1, 3, V).contiguous().cuda().expand(n, 3, V)
        dl = d.expand(1, 3, V).contiguous().cuda().expand(n, 3, V) if with_draft else None
        path, count, nxt = ops.verify_tree(lg, tokens, par.cuda(), u, 1.0, dl)
        first = torch.where(count > 1, tokens.gather(1, path[:, 1:2].clamp_min(0).long())[:, 0], nxt)
        seen = torch.bincount(first.cpu(), minlength=V).double()
        assert float(((seen - want) ** 2 / want).sum()) < 33.7


def test_verify_does_not_depend_on_the_batch():
    from torchplusplus_b200 import ops
    g = torch.Generator().manual_seed(12)
    logits, tokens, par, u, d = (x.cuda() for x in verify_inputs(g, 24, 7, 9001, BF16, True, True))
    all_ = ops.verify_tree(logits, tokens, par, u, 1.0, d)
    for b in (0, 5, 23):
        one = ops.verify_tree(*(x[b:b + 1].clone() for x in (logits, tokens, par, u)), 1.0,
                              d[b:b + 1, :6].clone())
        assert all(torch.equal(x[b:b + 1], y) for x, y in zip(all_, one))


def test_verify_uniforms_outside_the_unit_interval_are_its_ends():
    from torchplusplus_b200 import ops
    lg = torch.randn(4, 1, 3000, device="cuda")
    lg[:, :, :5] = -math.inf
    tok = torch.zeros(4, 1, dtype=torch.int64, device="cuda")
    par = torch.full((1,), -1, dtype=torch.int32, device="cuda")
    u = torch.tensor([[-1.0], [0.0], [1.0], [7.0]], device="cuda")
    nxt = ops.verify_tree(lg, tok, par, u)[2].tolist()
    assert nxt[0] == 5 and nxt[1] == 5 and nxt[2] == 2999 and nxt[3] == 2999


def test_verify_refusals():
    from torchplusplus_b200 import TppError, ops
    lg = torch.zeros(2, 3, 50, device="cuda")
    tok = torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    par = torch.tensor([-1, 0, 1], dtype=torch.int32, device="cuda")
    u = torch.zeros(2, 3, device="cuda")
    ops.verify_tree(lg, tok, par, u)
    for args, err in (((lg.cpu(), tok, par, u), RuntimeError), ((lg[0], tok, par, u), ValueError),
                      ((lg, tok.int(), par, u), ValueError), ((lg, tok, par.long(), u), ValueError),
                      ((lg, tok, par), ValueError), ((lg, tok, par, u.half()), ValueError),
                      ((lg, tok, par, u, -1.0), TppError), ((lg, tok, par, u, math.nan), TppError),
                      ((lg, tok, par, u, 1.0, lg.half()), TypeError),
                      ((lg, tok, par, u, 1.0, lg[:, :1]), ValueError),
                      ((lg.double(), tok, par, u), TypeError)):
        with pytest.raises(err):
            ops.verify_tree(*args)


# ------------------------------------------------------------------ commit
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("L,B,T,Hkv,D", [(1, 1, 1, 1, 8), (3, 4, 9, 2, 64), (2, 3, 70, 8, 128),
                                         (28, 2, 5, 1, 24)])
def test_commit(L, B, T, Hkv, D, paged, dtype):
    from torchplusplus_b200 import ops
    g = torch.Generator().manual_seed(T)
    cap = 192
    kt, vt = (torch.randn(L, B, T, Hkv, 2 * D, generator=g).to(dtype).cuda()[..., :D] for _ in "kv")
    count = torch.randint(0, T + 1, (B,), generator=g).int()
    count[0] = T
    path = torch.full((B, T), -1, dtype=torch.int32)
    for b in range(B):
        n = int(count[b])
        path[b, :n] = torch.randperm(T, generator=g)[:n].sort()[0].int()
    ctx = torch.randint(0, cap - T, (B,), generator=g).int()
    ctx[-1] = cap - T // 2 - 1        # the last rows are past the cache: skipped
    table = None
    if paged:
        table = torch.randperm(B * 3 + 2, generator=g)[:B * 3].view(B, 3).int()
        shape = (L, B * 3 + 2, Hkv, 64, D)
    else:
        shape = (L, B, Hkv, cap, D)
    kc, vc = (torch.randn(shape, generator=g).to(dtype).cuda() for _ in "kv")
    want = [kc.clone(), vc.clone()]
    for x, src in zip(want, (kt, vt)):
        for b in range(B):
            for i in range(int(count[b])):
                row = int(ctx[b]) + i
                if row >= cap:
                    continue
                if paged:
                    x[:, int(table[b, row // 64]), :, row % 64] = src[:, b, int(path[b, i])]
                else:
                    x[:, b, :, row] = src[:, b, int(path[b, i])]
    ops.kv_commit(kt, vt, path.cuda(), count.cuda(), ctx.cuda(), kc, vc,
                  block_table=None if table is None else table.cuda())
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])


def test_commit_ignores_nodes_and_blocks_that_are_none_and_refuses():
    from torchplusplus_b200 import ops
    kt = torch.randn(1, 1, 4, 1, 64, device="cuda").half()
    path = torch.tensor([[0, -1, 9, 3]], dtype=torch.int32, device="cuda")
    n = torch.tensor([100], dtype=torch.int32, device="cuda")          # more than T: T
    ctx = torch.tensor([62], dtype=torch.int32, device="cuda")
    pool = torch.zeros(1, 2, 1, 64, 64, device="cuda").half()
    vpool = pool.clone()
    table = torch.tensor([[1, 5]], dtype=torch.int32, device="cuda")   # block 5 is none
    ops.kv_commit(kt, kt, path, n, ctx, pool, vpool, table)
    want = torch.zeros_like(pool)
    want[0, 1, 0, 62] = kt[0, 0, 0, 0]
    assert torch.equal(pool, want) and torch.equal(vpool, want)
    c = torch.zeros(1, 1, 1, 64, 64, device="cuda").half()
    for args, err in (((kt.cpu(), kt, path, n, ctx, c, c), RuntimeError),
                      ((kt[0], kt[0], path, n, ctx, c, c), ValueError),
                      ((kt, kt, path.long(), n, ctx, c, c), ValueError),
                      ((kt, kt, path, n, ctx, c[:, :, :, :, :32], c), ValueError),
                      ((kt, kt, path, n, ctx, c.float(), c.float()), TypeError),
                      ((kt, kt, path, n, ctx, c.expand(1, 2, 1, 64, 64), c.expand(1, 2, 1, 64, 64)),
                       ValueError)):
        with pytest.raises(err):
            ops.kv_commit(*args)
