"""Packed-prompt operators (q/k norm + RoPE + cache rows, attention) against their
definitions in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
UNIT = {BF16: 2.0 ** -8, F16: 2.0 ** -11}  # half a step, relative


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def packed(lens, head=0, tail=0):
    """cu_seqlens (on the device) and the number of rows, with rows of no sequence
    before and behind."""
    cu = torch.tensor([0] + list(lens)).cumsum(0) + head
    return cu.to(torch.int32).cuda(), int(cu[-1]) + tail


# ------------------------------------------------------------------ attention
def attention_oracle(q, k, v, cu, causal=True, window=-1, scale=None):
    """Output and tolerance, both [N, Hq, D] in 64 bits (rows of no sequence: 0).

    Tolerance: the probabilities and the output are rounded once each to the storage
    type (u each, relative; a = sum w |v| bounds what the first does to the sum; f16
    weights below 2^-24 of the largest vanish, 2^-25 each); a score is a sum of D
    products in 32 bits, so its error is at most (D + 8) 2^-23 of the sum of their magnitudes, and it
    moves each weight by that, relative; 2^-19 covers the exponential, its argument's rounding
    against a maximum of up to 2^5 and the sums over the keys in 32 bits."""
    N, Hq, D = q.shape
    G, u = Hq // k.shape[1], UNIT[q.dtype]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(N, Hq, D, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    for a, b in zip(cu.tolist()[:-1], cu.tolist()[1:]):
        n = b - a
        if n == 0:
            continue
        far = torch.arange(n, device="cuda")[:, None] - torch.arange(n, device="cuda")
        hide = torch.zeros(n, n, dtype=torch.bool, device="cuda")
        if causal:
            hide |= far < 0
        if window >= 0:
            hide |= far > window
        for h in range(Hq):
            x, kk, vv = q[a:b, h].double(), k[a:b, h // G].double(), v[a:b, h // G].double()
            s = (x @ kk.T * scale).masked_fill(hide, -math.inf)
            big = (x.abs() @ kk.abs().T * abs(scale)).masked_fill(hide, 0).amax(1, keepdim=True)
            w = torch.softmax(s, 1)
            out[a:b, h] = o = w @ vv
            m = w @ vv.abs()
            tol[a:b, h] = u * (m + o.abs()) + (2 * (D + 8) * 2.0 ** -23 * big + 2.0 ** -19) * m \
                + 2.0 ** -24
            if q.dtype is F16:
                tol[a:b, h] += n * 2.0 ** -25 * vv.abs().amax()
    return out, tol


def check_attention(q, k, v, cu, got=None, **kw):
    from torchplusplus_b200 import ops
    got = ops.attention_packed(q, k, v, cu, causal=kw.get("causal", True),
                               window_left=kw.get("window", -1),
                               scale=kw.get("scale")) if got is None else got
    ref, tol = attention_oracle(q, k, v, cu, **kw)
    rows = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
    rows[int(cu[0]):int(cu[-1])] = True
    bad = ((got.double() - ref).abs() > tol) | ~got.double().isfinite()
    assert not bad[rows].any(), (bad[rows].sum().item(),
                                 ((got.double() - ref).abs() / tol)[rows].max().item())
    return got


def operands(seed, N, Hq, Hkv, D, dtype, spread=2.0):
    g = gen(seed)
    return (randn(g, N, Hq, D, dtype=dtype) * spread, randn(g, N, Hkv, D, dtype=dtype),
            randn(g, N, Hkv, D, dtype=dtype))


@pytest.mark.parametrize("lens", [[1], [2], [127], [128], [129], [300], [1, 1, 1], [0, 5, 0, 129, 0],
                                  [64, 65, 63], [256, 257], [500, 1, 77, 260]])
@pytest.mark.parametrize("Hq,Hkv,D,dtype", [(4, 2, 128, BF16), (4, 4, 128, F16), (3, 1, 64, BF16),
                                            (8, 1, 64, F16), (14, 2, 128, BF16)])
def test_attention_of_lengths(lens, Hq, Hkv, D, dtype):
    cu, N = packed(lens)
    check_attention(*operands(1, N, Hq, Hkv, D, dtype), cu)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [-1, 0, 1, 63, 127, 128, 129, 300, 1 << 40])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 2, 128), (5, 1, 64)])
def test_attention_windows(causal, window, Hq, Hkv, D):
    cu, N = packed([700, 3, 130, 385])
    check_attention(*operands(2, N, Hq, Hkv, D, BF16), cu, causal=causal, window=window)


@pytest.mark.parametrize("Hq,Hkv", [(128, 1), (100, 1), (43, 1), (64, 1), (17, 1), (32, 8), (6, 6)])
def test_attention_group_sizes(Hq, Hkv):
    cu, N = packed([1, 40, 150])
    check_attention(*operands(3, N, Hq, Hkv, 64, BF16), cu)


@pytest.mark.parametrize("Hq,Hkv,D,dtype", [(4, 2, 128, BF16), (2, 2, 64, F16), (7, 1, 128, F16)])
def test_attention_long(Hq, Hkv, D, dtype):
    cu, N = packed([4100, 1, 2049])
    check_attention(*operands(4, N, Hq, Hkv, D, dtype), cu)


@pytest.mark.parametrize("seed,n", [(5, 31), (6, 33), (7, 700), (8, 3000)])
def test_attention_many_sequences(seed, n):
    lens = torch.randint(0, 200 if n < 100 else 40 if n < 1000 else 5, (n,),
                         generator=torch.Generator().manual_seed(seed)).tolist()
    cu, N = packed(lens)
    check_attention(*operands(seed, N, 4, 2, 64, BF16), cu)


def test_attention_fills_every_cta_several_times():
    cu, N = packed([600, 1200, 333, 901, 64] * 4)
    check_attention(*operands(8, N, 16, 8, 128, BF16), cu)


def test_attention_growing_scores():
    """Scores that grow along the keys move every row's maximum at every tile."""
    cu, N = packed([1000])
    q, k, v = operands(9, N, 2, 1, 128, BF16, 0.1)
    q[..., 0] = 3.0
    k[..., 0] = (torch.arange(N, device="cuda")[:, None] / 8).to(BF16)
    check_attention(q, k, v, cu)
    k[..., 0] = -k[..., 0]
    check_attention(q, k, v, cu)


@pytest.mark.parametrize("scale", [-0.07, 0.0, 1.0])
def test_attention_scales(scale):
    cu, N = packed([200, 131])
    check_attention(*operands(10, N, 4, 2, 64, F16, 0.5), cu, scale=scale)


def test_attention_views_and_rows_of_no_sequence():
    """Operands by strides; rows before the first and behind the last sequence hold NaN,
    and their outputs stay as they were."""
    from torchplusplus_b200 import ops
    Hq, Hkv, D = 6, 2, 128
    cu, N = packed([150, 20, 0, 257], head=9, tail=70)
    g = gen(11)
    qkv = randn(g, N, (Hq + 2 * Hkv) * D, dtype=BF16)
    qkv[:9] = math.nan
    qkv[N - 70:] = math.inf
    q = qkv[:, :Hq * D].view(N, Hq, D)
    k = qkv[:, Hq * D:(Hq + Hkv) * D].view(N, Hkv, D)
    v = qkv[:, (Hq + Hkv) * D:].view(N, Hkv, D)
    room = torch.full((N, Hq + 1, D), 7.0, dtype=BF16, device="cuda")
    out = room[:, 1:]
    got = ops.attention_packed(q, k, v, cu, out=out)
    assert got is out
    check_attention(q, k, v, cu, got=got)
    assert (room[:, 0] == 7).all() and (room[:9] == 7).all() and (room[N - 70:] == 7).all()
    # a row stride that only allows 16-byte stores
    odd = torch.full((N, Hq * D + 8), 7.0, dtype=BF16, device="cuda")
    got = ops.attention_packed(q, k, v, cu, out=odd[:, 8:].view(N, Hq, D))
    check_attention(q, k, v, cu, got=got)
    assert (odd[:, :8] == 7).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("causal,window", [(True, -1), (True, 40), (False, -1)])
def test_attention_non_finite_values(D, bad, causal, window):
    """A non-finite V element reaches the rows that see it, in its dimension, and no others."""
    cu, N = packed([130, 300, 90])
    q, k, v = operands(12, N, 4, 2, D, BF16, 0.5)
    clean = v.clone()
    at = [(130 + 5, 0, 3), (130 + 128, 1, D - 1), (130 + 299, 0, 40), (129, 1, 0)]
    for r, h, d in at:
        v[r, h, d] = bad
        clean[r, h, d] = 0
    from torchplusplus_b200 import ops
    got = ops.attention_packed(q, k, v, cu, causal=causal, window_left=window).double()
    ref, tol = attention_oracle(q, k, clean, cu, causal=causal, window=window)
    hit = torch.zeros_like(got, dtype=torch.bool)
    row = torch.arange(N, device="cuda")
    seq = torch.bucketize(row, cu[1:].long(), right=True)
    for r, h, d in at:
        sees = seq == seq[r]
        if causal:
            sees &= row >= r
        if window >= 0:
            sees &= row - r <= window
        hit[sees, 2 * h:2 * h + 2, d] = True
    assert ((got - ref).abs() <= tol)[~hit].all()
    if bad != bad:
        assert got[hit].isnan().all()
    else:
        assert (got[hit] == bad).all() or not got[hit].isfinite().any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 30, 90])
def test_attention_non_finite_values_in_every_sequence(n, D):
    """Many short sequences a CTA: what one's V holds is known when its rows are written."""
    B = 4000
    cu, N = packed([n] * B)
    q, k, v = operands(22, N, 4, 2, D, BF16, 0.5)
    at = torch.arange(B, device="cuda") * n + n // 2
    v[at, :, 7] = math.inf
    from torchplusplus_b200 import ops
    got = ops.attention_packed(q, k, v, cu).view(B, n, 4, D)
    assert (got[:, n // 2:, :, 7] == math.inf).all()
    assert got[:, :n // 2, :, 7].isfinite().all()
    assert got[..., :7].isfinite().all() and got[..., 8:].isfinite().all()


def test_attention_non_finite_keys_stay_hidden():
    cu, N = packed([100, 200])
    q, k, v = operands(13, N, 2, 2, 128, BF16)
    from torchplusplus_b200 import ops
    want = ops.attention_packed(q, k, v, cu)
    k[150, 0, 5] = math.nan
    k[99, 1, 0] = math.inf
    got = ops.attention_packed(q, k, v, cu)
    assert torch.equal(got[:99], want[:99]) and torch.equal(got[100:150], want[100:150])
    assert torch.equal(got[150:, 1], want[150:, 1])
    assert got[150:, 0].isnan().all()


def test_attention_on_a_side_stream_and_in_a_graph():
    from torchplusplus_b200 import ops
    cu, N = packed([100, 333, 64])
    q, k, v = operands(14, N, 4, 2, 128, BF16)
    want = ops.attention_packed(q, k, v, cu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a = ops.attention_packed(q, k, v, cu)
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.current_stream().wait_stream(s)
    with torch.cuda.graph(graph):
        ops.attention_packed(q, k, v, cu, out=out)
    graph.replay()
    assert torch.equal(a, want) and torch.equal(out, want)
    # other lengths and other values in the same buffers
    cu.copy_(torch.tensor([0, 300, 301, 480], dtype=torch.int32))
    q.mul_(0.5)
    out.zero_()
    graph.replay()
    check_attention(q, k, v, cu, got=out)
    assert (out[480:] == 0).all()


@pytest.mark.parametrize("Hq,Hkv", [(4, 2), (6, 2)])
def test_attention_into_its_queries(Hq, Hkv):
    from torchplusplus_b200 import ops
    cu, N = packed([300, 5, 131])
    q, k, v = operands(16, N, Hq, Hkv, 64, BF16)
    want = ops.attention_packed(q, k, v, cu)
    assert ops.attention_packed(q, k, v, cu, out=q) is q and torch.equal(q, want)


def test_attention_of_lengths_that_do_not_ascend():
    """Whatever cu_seqlens holds, only rows of q, k and v are read and rows of out written."""
    from torchplusplus_b200 import ops
    q, k, v = operands(17, 400, 4, 2, 128, BF16)
    out = torch.zeros(420, 4, 128, dtype=BF16, device="cuda")
    cu = torch.tensor([-5, 100, 50, 1 << 30, -(1 << 31), 20, 500], dtype=torch.int32, device="cuda")
    ops.attention_packed(q, k, v, cu, out=out[:400])
    assert (out[400:] == 0).all() and ops.device_error() == 0
    # [0, 100), none, [50, 400), none, [0, 20) and [20, 400): the rows of no two of them
    cos = torch.ones(400, 128, device="cuda")
    qkv = torch.randn(400, 8 * 128, generator=gen(17), device="cuda").to(BF16)
    kc = torch.zeros(6, 2, 64, 128, dtype=BF16, device="cuda")
    ops.qk_norm_rope_packed(qkv, None, None, 1e-6, cos, cos, cu, 4, 2, kc, kc.clone())
    torch.cuda.synchronize()


def test_attention_of_no_rows():
    from torchplusplus_b200 import ops
    q, k, v = operands(15, 0, 4, 2, 128, BF16)
    assert ops.attention_packed(q, k, v, torch.zeros(1, dtype=torch.int32, device="cuda")).shape \
        == (0, 4, 128)
    q, k, v = operands(15, 40, 4, 2, 128, BF16)
    out = torch.full_like(q, 3)
    for cu in ([0], [0, 0, 0], [40, 40]):
        ops.attention_packed(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), out=out)
    assert (out == 3).all()
    assert ops.device_error() == 0


# ------------------------------------------------------------------ norm, positions, cache
def rope_oracle(qkv, qn, kn, eps, cos, sin, cu, Hq, Hkv):
    """q, k and their tolerances in 64 bits; the sequence and position of each row (-1: none)."""
    N, D = qkv.shape[0], qkv.shape[1] // (Hq + 2 * Hkv)
    seq = torch.full((N,), -1, device="cuda")
    pos = torch.zeros(N, dtype=torch.int64, device="cuda")
    for b, (s, e) in enumerate(zip(cu.tolist()[:-1], cu.tolist()[1:])):
        seq[s:e], pos[s:e] = b, torch.arange(e - s, device="cuda")
    inside = (pos < cos.shape[0])[:, None, None]
    at = pos.clamp_max(cos.shape[0] - 1)
    c, s = cos.double()[at][:, None], sin.double()[at][:, None]
    out = []
    x = qkv.double().view(N, Hq + 2 * Hkv, D)
    for part, w in ((x[:, :Hq], qn), (x[:, Hq:Hq + Hkv], kn)):
        if w is not None:
            part = part * (part.pow(2).mean(-1, keepdim=True) + eps).rsqrt() * w.double()
        half = torch.cat([-part[..., D // 2:], part[..., :D // 2]], -1)
        y = torch.where(inside, part * c + half * s, 0)
        # one rounding to the type; a sum of D squares, its root and five products in 32 bits
        mag = (part.abs() * c.abs() + half.abs() * s.abs())
        out += [y, UNIT[qkv.dtype] * y.abs() + (D / 2 + 16) * 2.0 ** -24 * mag + 2.0 ** -25]
    return out, seq, pos


@pytest.mark.parametrize("cache", ["none", "rows", "paged"])
@pytest.mark.parametrize("lens,head,tail", [([1], 0, 0), ([5, 0, 64, 65], 3, 4), ([700, 900, 31], 0, 5)])
@pytest.mark.parametrize("Hq,Hkv,D,dtype,cs,norm", [
    (4, 2, 128, BF16, F16, True), (7, 1, 64, F16, BF16, True), (5, 5, 16, BF16, F32, True),
    (3, 3, 32, F16, F16, False), (8, 2, 256, BF16, F16, True)])
def test_rope_packed(cache, lens, head, tail, Hq, Hkv, D, dtype, cs, norm):
    from torchplusplus_b200 import ops
    cu, N = packed(lens, head, tail)
    g = gen(20)
    qkv = randn(g, N, (Hq + 2 * Hkv) * D + 8, dtype=dtype)[:, :-8]
    qn = (1 + 0.2 * randn(g, D)).to(dtype) if norm else None
    kn = (1 + 0.2 * randn(g, D)).to(dtype) if norm else None
    ang = torch.rand(max(lens), D, generator=g, device="cuda") * 6
    cos, sin = ang.cos().to(cs), ang.sin().to(cs)
    B, cols = len(lens), -(-max(lens) // 64) + 1
    kc = vc = table = None
    if cache == "rows":
        kc, vc = randn(g, B, Hkv, max(lens) + 3, D, dtype=dtype), randn(g, B, Hkv, max(lens) + 3, D, dtype=dtype)
    elif cache == "paged":
        kc, vc = randn(g, B * cols, Hkv, 64, D, dtype=dtype), randn(g, B * cols, Hkv, 64, D, dtype=dtype)
        table = torch.randperm(B * cols, generator=g, device="cuda").view(B, cols).to(torch.int32)
    want = None if kc is None else (kc.clone(), vc.clone())
    q0 = torch.full((N, Hq, D), 9.0, dtype=dtype, device="cuda")
    k0 = torch.full((N, Hkv, D), 9.0, dtype=dtype, device="cuda")
    q, k = ops.qk_norm_rope_packed(qkv, qn, kn, 1e-6, cos, sin, cu, Hq, Hkv, k_cache=kc, v_cache=vc,
                                   block_table=table, q_out=q0, k_out=k0)
    (qr, qt, kr, kt), seq, pos = rope_oracle(qkv, qn, kn, 1e-6, cos, sin, cu, Hq, Hkv)
    has = seq >= 0
    assert ((q.double() - qr).abs() <= qt)[has].all() and ((k.double() - kr).abs() <= kt)[has].all()
    assert (q[~has] == 9).all() and (k[~has] == 9).all()
    if kc is not None:
        v = qkv[:, (Hq + Hkv) * D:].view(N, Hkv, D)
        b, at = seq[has], pos[has]
        if table is not None:
            b, at = table.long()[b, at // 64], at % 64
        want[0][b, :, at], want[1][b, :, at] = k[has], v[has]
        assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])


def test_rope_packed_outside_tables_and_cache():
    """Positions beyond the tables give zero rows; rows beyond the cache or of blocks
    outside the pools are skipped."""
    from torchplusplus_b200 import ops
    Hq, Hkv, D = 2, 2, 64
    cu, N = packed([200, 70])
    g = gen(21)
    qkv = randn(g, N, (Hq + 2 * Hkv) * D, dtype=BF16)
    qkv[150] = 0
    w = torch.ones(D, dtype=BF16, device="cuda")
    cos, sin = torch.ones(100, D, device="cuda"), torch.zeros(100, D, device="cuda")
    kc, vc = (torch.full((2, Hkv, 130, D), 5.0, dtype=BF16, device="cuda") for _ in range(2))
    q, k = ops.qk_norm_rope_packed(qkv, w, w, 0.0, cos, sin, cu, Hq, Hkv, kc, vc)
    assert (q[100:200] == 0).all() and (k[100:200] == 0).all() and k[:100].abs().amin(2).amax() > 0
    assert torch.equal(vc[0].transpose(0, 1), qkv[:130, 2 * Hkv * D:].view(130, Hkv, D))
    assert (vc[1, :, 70:] == 5).all() and (kc[1, :, 70:] == 5).all()
    pool = torch.full((3, Hkv, 64, D), 5.0, dtype=BF16, device="cuda")
    pv = pool.clone()
    table = torch.tensor([[1, -1, 7], [2, 3, 0]], dtype=torch.int32, device="cuda")
    ops.qk_norm_rope_packed(qkv, None, None, 0.0, cos, sin, cu, Hq, Hkv, pool, pv, table)
    assert torch.equal(pv[1].transpose(0, 1), qkv[:64, 2 * Hkv * D:].view(64, Hkv, D))
    assert torch.equal(pv[2].transpose(0, 1), qkv[200:264, 2 * Hkv * D:].view(64, Hkv, D))
    assert (pv[0] == 5).all() and (pool[0] == 5).all()


def test_packed_prefill_together():
    """A projection's rows through both operators, the cache then read by decode attention."""
    from torchplusplus_b200 import ops
    Hq, Hkv, D = 8, 4, 128
    lens = [33, 1, 190, 64]
    cu, N = packed(lens)
    g = gen(22)
    qkv = randn(g, N, (Hq + 2 * Hkv) * D, dtype=BF16)
    ang = torch.rand(200, D // 2, generator=g, device="cuda").repeat(1, 2) * 6
    cos, sin = ang.cos().half(), ang.sin().half()
    kc, vc = (torch.zeros(4, Hkv, 256, D, dtype=BF16, device="cuda") for _ in range(2))
    q, k = ops.qk_norm_rope_packed(qkv, None, None, 1e-6, cos, sin, cu, Hq, Hkv, kc, vc)
    v = qkv[:, (Hq + Hkv) * D:].view(N, Hkv, D)
    o = check_attention(q, k, v, cu)
    last = cu[1:].long() - 1
    dec = ops.attention_decode(q[last], kc, vc, torch.tensor(lens, dtype=torch.int32, device="cuda"), 190)
    _, tol = attention_oracle(q, k, v, cu)
    assert ((dec.double() - o[last].double()).abs() <= 2 * tol[last]).all()


# ------------------------------------------------------------------ refusals
def test_refusals():
    from torchplusplus_b200 import TppError, ops
    cu, N = packed([20])
    q, k, v = operands(30, N, 4, 2, 128, BF16)
    bad = [
        (TypeError, lambda: ops.attention_packed(q.float(), k.float(), v.float(), cu)),
        (TypeError, lambda: ops.attention_packed(q, k, v.half(), cu)),
        (ValueError, lambda: ops.attention_packed(q[:, :3], k, v, cu)),
        (ValueError, lambda: ops.attention_packed(q[:19], k, v, cu)),
        (ValueError, lambda: ops.attention_packed(q, k, v, cu.long())),
        (ValueError, lambda: ops.attention_packed(q, k, v, cu[:0])),
        (RuntimeError, lambda: ops.attention_packed(q, k, v, cu.cpu())),
        (ValueError, lambda: ops.attention_packed(q, k, v, cu, out=q[:10])),
        (ValueError, lambda: ops.attention_packed(q, k, v, cu, out=q[:1].expand(N, -1, -1))),
        (TppError, lambda: ops.attention_packed(*operands(1, N, 2, 2, 96, BF16), cu)),
        (TppError, lambda: ops.attention_packed(*operands(1, N, 129, 1, 64, BF16), cu)),
        (TppError, lambda: ops.attention_packed(q, k, v, cu, scale=math.inf)),
    ]
    qkv = torch.zeros(N, 8 * 128, dtype=BF16, device="cuda")
    t = torch.zeros(30, 128, device="cuda")
    kc = torch.zeros(1, 2, 64, 128, dtype=BF16, device="cuda")

    def rope(x=qkv, **kw):
        return ops.qk_norm_rope_packed(x, None, None, 1e-6, t, t, cu, 4, 2, **kw)
    bad += [
        (ValueError, lambda: rope(qkv[:, :-1])),
        (ValueError, lambda: rope(k_cache=kc)),
        (ValueError, lambda: rope(block_table=cu[None])),
        (ValueError, lambda: rope(k_cache=kc[:, :1], v_cache=kc[:, :1])),
        (ValueError, lambda: rope(k_cache=kc.expand(2, -1, -1, -1), v_cache=kc.expand(2, -1, -1, -1))),
        (TypeError, lambda: rope(k_cache=kc.half(), v_cache=kc.half())),
    ]
    for err, call in bad:
        with pytest.raises(err):
            call()
    assert ops.device_error() == 0


def test_all_operators_on_two_streams_at_once():
    """Calls that overlap on the device give what they give one after another."""
    from torchplusplus_b200 import ops
    cu, N = packed([700, 3, 1500, 64])
    q, k, v = operands(31, N, 16, 8, 128, BF16)
    g = gen(32)
    qkv, w = randn(g, N, 32 * 128, dtype=BF16), randn(g, 128, dtype=BF16)
    cos, sin = randn(g, 1500, 128), randn(g, 1500, 128)
    x, head = randn(g, 300, 1024, dtype=BF16), randn(g, 30001, 1024, dtype=BF16) / 32
    tok = torch.randint(0, 30001, (300,), generator=g, device="cuda")
    logits = randn(g, 300, 30001, dtype=BF16)
    calls = [lambda: (ops.attention_packed(q, k, v, cu),),
             lambda: ops.qk_norm_rope_packed(qkv, w, w, 1e-6, cos, sin, cu, 16, 8),
             lambda: ops.linear_logprobs(x, head, tok),
             lambda: ops.token_logprobs(logits, tok, top=20)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for turn in range(12):
        for at, st in enumerate(streams):
            with torch.cuda.stream(st):
                n = (turn + at * (1 + turn // 4)) % 4
                got.append((n, calls[n]()))
    torch.cuda.synchronize()
    for n, out in got:
        assert all(torch.equal(a, b) for a, b in zip(out, want[n])), n
    assert ops.device_error() == 0
