"""Packed-prompt operators at the edges of what their documentation allows, against their
definitions in 64 bits."""
import math

import pytest
import torch

from .test_logprobs_gpu import check, check_head, operands as head_operands
from .test_packed_gpu import (BF16, F16, F32, attention_oracle, check_attention, gen, packed, randn,
                              rope_oracle)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ norm, positions, cache
def check_rope(lens, head, tail, Hq, Hkv, D, dtype, cache, norm):
    from torchplusplus_b200 import ops
    cu, N = packed(lens, head, tail)
    g = gen(40)
    qkv = randn(g, N, (Hq + 2 * Hkv) * D, dtype=dtype)
    qn = (1 + 0.2 * randn(g, D)).to(dtype) if "q" in norm else None
    kn = (1 + 0.2 * randn(g, D)).to(dtype) if "k" in norm else None
    ang = torch.rand(max(lens), D, generator=g, device="cuda") * 6
    cos, sin = ang.cos().half(), ang.sin().half()
    B, cols = len(lens), -(-max(lens) // 64)
    kc = vc = table = want = None
    if cache == "rows":
        kc, vc = (randn(g, B, Hkv, max(lens), D, dtype=dtype) for _ in range(2))
    elif cache == "paged":
        kc, vc = (randn(g, B * cols, Hkv, 64, D, dtype=dtype) for _ in range(2))
        table = torch.randperm(B * cols, generator=g, device="cuda").view(B, cols).to(torch.int32)
    if kc is not None:
        want = kc.clone(), vc.clone()
    q = torch.full((N, Hq, D), 9.0, dtype=dtype, device="cuda")
    k = torch.full((N, Hkv, D), 9.0, dtype=dtype, device="cuda")
    ops.qk_norm_rope_packed(qkv, qn, kn, 1e-6, cos, sin, cu, Hq, Hkv, k_cache=kc, v_cache=vc,
                            block_table=table, q_out=q, k_out=k)
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


@pytest.mark.parametrize("norm", ["q", "k", "qk", ""])
@pytest.mark.parametrize("cache", ["none", "rows", "paged"])
@pytest.mark.parametrize("Hq,Hkv,D,dtype", [(4, 2, 128, BF16), (3, 1, 64, F16), (5, 3, 32, BF16),
                                            (2, 2, 256, F16), (3, 2, 16, BF16)])
def test_rope_of_either_norm(norm, cache, Hq, Hkv, D, dtype):
    check_rope([5, 0, 64, 66], 3, 4, Hq, Hkv, D, dtype, cache, norm)


# From N (Hq + Hkv, 2 Hkv with a cache) D / 16 = 4 * 2048 * 148 on a unit of lanes takes four
# heads; these group sizes leave it one, two, three or all four of its last ones.
@pytest.mark.parametrize("norm", ["q", "k", "qk", ""])
@pytest.mark.parametrize("cache", ["none", "rows", "paged"])
@pytest.mark.parametrize("Hq,Hkv,D,dtype", [(7, 3, 128, BF16), (8, 2, 128, F16), (5, 1, 256, BF16),
                                            (14, 4, 64, F16)])
def test_rope_of_many_rows(norm, cache, Hq, Hkv, D, dtype):
    rows = -(-4 * 2048 * 160 * 16 // ((Hq + Hkv * (1 if cache == "none" else 2)) * D))
    lens = [rows // 2, 1, rows // 3, 0, 130]
    lens.append(rows - sum(lens) + 37)
    check_rope(lens, 2, 3, Hq, Hkv, D, dtype, cache, norm)


# ------------------------------------------------------------------ scores
@pytest.mark.parametrize("step", [8, 24, 56])
@pytest.mark.parametrize("which", ["x", "weight"])
def test_head_of_rows_that_overlap(which, step):
    """A row stride below the rows' length (a view of a signal's windows)."""
    from torchplusplus_b200 import ops
    g = gen(41)
    N, V, E = 33, 150, 64
    rows = dict(x=N, weight=V)
    got = dict(x=randn(g, N, E, dtype=BF16), weight=randn(g, V, E, dtype=BF16))
    room = randn(g, (rows[which] - 1) * step + E, dtype=BF16)
    got[which] = room.as_strided((rows[which], E), (step, 1))
    tok = torch.randint(0, V, (N,), generator=g, device="cuda")
    out = ops.linear_logprobs(got["x"], got["weight"], tok)
    got[which] = got[which].contiguous()
    want = ops.linear_logprobs(got["x"], got["weight"], tok)
    assert all(torch.equal(a, b) for a, b in zip(out, want))


# ------------------------------------------------------------------ single rows at any pitch
def pitched(g, rows, *shape, dtype=BF16):
    """Rows of `shape` at a pitch that is no multiple of 16 bytes."""
    n = torch.Size(shape).numel()
    return randn(g, rows, n + 5, dtype=dtype)[:, :n].view(rows, *shape)


def test_single_rows_at_any_pitch():
    from torchplusplus_b200 import ops
    g = gen(42)
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    x, w = pitched(g, 3, 64)[:1], pitched(g, 3, 64)[:1]
    tok = torch.zeros(1, dtype=torch.int64, device="cuda")
    out = ops.linear_logprobs(x, w, tok)
    assert out[0].item() == 0 and out[1].item() == 0  # one token: certain
    q, k, v, o = (pitched(g, 2, h, 64)[:1] for h in (4, 2, 2, 4))
    rest = o.untyped_storage()[-2 * (4 * 64 + 10):].tolist()
    assert ops.attention_packed(q, k, v, cu, out=o) is o
    assert torch.equal(o, v.repeat_interleave(2, 1)) and o.untyped_storage()[-2 * (4 * 64 + 10):].tolist() == rest
    t = randn(g, 8, 64)
    qkv = pitched(g, 2, 8 * 64)[:1]
    kc, vc = pitched(g, 2, 2, 8, 64)[:1], pitched(g, 2, 2, 8, 64)[:1]
    want = kc.clone(), vc.clone()
    got = ops.qk_norm_rope_packed(qkv, None, None, 1e-6, t, t, cu, 4, 2, kc, vc)
    ref = ops.qk_norm_rope_packed(qkv.clone(), None, None, 1e-6, t, t, cu, 4, 2, *want)
    for a, b in ((got[0], ref[0]), (got[1], ref[1]), (kc, want[0]), (vc, want[1])):
        assert torch.equal(a, b)
    assert ops.device_error() == 0


# Vocabularies that end inside a block of 16 logits, products of one chain and of several.
@pytest.mark.parametrize("E,V", [(64, 1003), (1024, 1003), (1024, 37), (520, 300)])
@pytest.mark.parametrize("temperature", [1e-6, 1e30, 1e37, 1e38, 1e39, 1e300])
def test_head_at_any_temperature(E, V, temperature):
    check_head(*head_operands(43, 40, E, V, BF16), temperature)


@pytest.mark.parametrize("E,V", [(64, 1003), (1024, 1003), (1024, 37), (520, 300)])
@pytest.mark.parametrize("size", [2.0 ** 50, 2.0 ** 58, 2.0 ** 60])
def test_head_of_large_logits(E, V, size):
    """Logits of up to some 2^122, both signs: their differences stay finite."""
    x, w, tok = head_operands(44, 40, E, V, BF16)
    check_head(x * size, w * size, tok)


def test_head_of_log_probabilities_next_to_the_largest_number():
    """A log probability of -3.2e38 is a float32, and 1.44 times it (in bits) is none."""
    from torchplusplus_b200 import ops
    x = torch.zeros(2, 8, dtype=BF16, device="cuda")
    w = torch.zeros(40, 8, dtype=BF16, device="cuda")
    x[:, 0] = 2.0 ** 63
    w[3, 0], w[5, 0] = 2.0 ** 63 * 1.875, -(2.0 ** 63) * 1.875
    tok = torch.tensor([5, 3], device="cuda")
    lp, ent = ops.linear_logprobs(x, w, tok)
    assert lp.tolist() == [-2.0 ** 127 * 1.875, 0.0] and ent.tolist() == [0.0, 0.0]
    lp, ent = ops.linear_logprobs(x, w, tok, temperature=2.0)
    assert lp.tolist() == [-2.0 ** 126 * 1.875, 0.0] and ent.tolist() == [0.0, 0.0]
    # and as far off at a temperature below 1
    lp, _ = ops.linear_logprobs(x / 2 ** 10, w, tok, temperature=2.0 ** -10)
    assert lp.tolist() == [-2.0 ** 127 * 1.875, 0.0]


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bits", [20.0, 25.2, 28.0])
def test_attention_f16_of_many_small_weights(D, bits, causal):
    """A first key of weight 1 (and value 0) before thousands of 2^-bits (and value 1): what
    each gives is below f16's smallest number, their sum is not.

    Tolerance: as the oracle's, but for what a weight loses below the smallest normal number:
    weights are held 2^7 times as large as against the row's largest, so 2^-32 each."""
    from torchplusplus_b200 import ops
    cu, N = packed([6000, 1, 500])
    q = torch.zeros(N, 4, D, dtype=F16, device="cuda")
    k = torch.zeros(N, 2, D, dtype=F16, device="cuda")
    v = torch.ones(N, 2, D, dtype=F16, device="cuda")
    q[:, :, 0] = 1
    for a in cu.tolist()[:-1]:
        k[a, :, 0], v[a] = bits * math.log(2), 0
    got = ops.attention_packed(q, k, v, cu, causal=causal, scale=1.0)
    ref, tol = attention_oracle(q, k, v, cu, causal=causal, scale=1.0)
    for a, b in zip(cu.tolist()[:-1], cu.tolist()[1:]):
        tol[a:b] -= (b - a) * (2.0 ** -25 - 2.0 ** -32)  # (of values of 1)
    assert ((got.double() - ref).abs() <= tol).all(), ((got.double() - ref).abs() / tol).max().item()


# 111 to 443 rows take two or four CTAs each, with 128 threads from 128 * 64 bytes a CTA on:
# noted hits and the join over the CTAs together.
@pytest.mark.parametrize("N,V", [(130, 33013), (221, 17011), (222, 17011), (300, 12007), (443, 9001)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_logprobs_of_rows_over_some_ctas(N, V, dtype):
    ix = torch.arange(V, device="cuda")
    low = torch.finfo(dtype).min
    rows = [
        torch.zeros(V),                                                    # all equal
        ix / V * 60 - 30, 30 - ix / V * 60,                                # in order
        torch.where(ix % 3 == 0, -math.inf, torch.where(ix % 37 == 5, 1.0, 0.0)),
        torch.where(ix < V - 2, -math.inf, 2.0),                           # two tokens left
        torch.where(ix < 5, 3.0 * (ix % 2), low),
        torch.full((V,), -math.inf),
        torch.where(ix == V // 2, math.nan, ix % 11),
        torch.where(ix == V - 1, math.inf, ix % 11),
        torch.where(ix % 2 == 0, 0.0, -0.0),
        torch.where(ix == V - 1, 60.0, ix % 13),
        torch.where((ix > V // 2) & (ix < V // 2 + 40), 9.0, ix % 5 * 1.0),  # across CTAs
    ]
    x = (torch.randn(N, V, generator=gen(45), device="cuda") * 3).to(dtype)
    for i, r in enumerate(rows):
        x[7 * i + 1] = r.to(device="cuda", dtype=dtype)
    tok = torch.randint(0, V, (N,), generator=gen(46), device="cuda")
    for top in (0, 1, 9, 32):
        check(x, tok, top=top)


@pytest.mark.parametrize("off,ld", [(3, 17019), (1, 17013)])
def test_logprobs_of_strided_rows_over_some_ctas(off, ld):
    room = (torch.randn(150, ld, generator=gen(47), device="cuda") * 3).to(BF16)
    check(room[:, off:off + 17011], torch.randint(0, 17011, (150,), generator=gen(48), device="cuda"), top=7)


# ------------------------------------------------------------------ lengths that make no sense
def guarded(*shape, value):
    """A tensor in the middle of a larger one full of `value`, and that one."""
    n = torch.Size(shape).numel()
    room = torch.full((n + 2 * 65536,), value, dtype=BF16, device="cuda")
    return room[65536:65536 + n].view(shape), room


def test_lengths_that_do_not_ascend_write_rows_only():
    """Whatever cu_seqlens holds, attention reads its spans cut to [0, N), and both operators
    write rows of their outputs and caches only."""
    from torchplusplus_b200 import ops
    N, Hq, Hkv, D = 400, 4, 2, 128
    g = gen(49)
    q, k, v = randn(g, N, Hq, D, dtype=BF16), randn(g, N, Hkv, D, dtype=BF16), randn(g, N, Hkv, D, dtype=BF16)
    qkv = randn(g, N, (Hq + 2 * Hkv) * D, dtype=BF16)
    cos = torch.ones(N, D, device="cuda")
    wild = [-7, 100, 60, 60, -9, -2, -(1 << 31), -5, 0, 0]    # rows 0 to 99 once
    late = [1 << 30, 500, 450, 250, 1 << 30, (1 << 31) - 1]   # rows 250 to 399 once
    for cu, a, b in ((wild, 0, 100), (late, 250, 400)):
        cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
        out, room = guarded(N, Hq, D, value=7.0)
        ops.attention_packed(q, k, v, cu, out=out)
        span = torch.tensor([a, b], dtype=torch.int32, device="cuda")
        ref, tol = attention_oracle(q, k, v, span)
        assert ((out.double() - ref).abs() <= tol)[a:b].all()
        out[a:b] = 7
        assert (room == 7).all() and ops.device_error() == 0
        # the norm and its cache: rows of its own outputs, and nothing else
        B = cu.shape[0] - 1
        got = [guarded(*s, value=7.0) for s in ((N, Hq, D), (N, Hkv, D), (B, Hkv, 64, D), (B, Hkv, 64, D))]
        ops.qk_norm_rope_packed(qkv, None, None, 1e-6, cos, cos, cu, Hq, Hkv, got[2][0], got[3][0],
                                q_out=got[0][0], k_out=got[1][0])
        for t, room in got:
            t.fill_(7)
            assert (room == 7).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("power", [19, 21, 23, 24, 25, 26])
def test_attention_of_large_scores(D, power, dtype):
    """Scores of 2^19 to 2^26 (in bits) whose maximum grows by up to 8 from step to step: where a
    float32 ends at whole numbers, weights stay finite in the storage type."""
    cu, N = packed([300, 40])
    for grow in (4, 8):
        q = torch.zeros(N, 2, D, dtype=dtype, device="cuda")
        k = torch.zeros(N, 1, D, dtype=dtype, device="cuda")
        q[:, :, 0], q[:, :, 1] = 2.0 ** (power - 13), 1
        k[:, :, 0] = 2.0 ** 13
        k[:, :, 1] = (64 + torch.arange(N, device="cuda") // 80 * grow).to(dtype)[:, None]
        v = randn(gen(50), N, 1, D, dtype=dtype)
        check_attention(q, k, v, cu, scale=math.log(2))
        check_attention(q, k, v, cu, scale=math.log(2), causal=False)
