"""Draft-tree operators where their plans, arguments and inputs leave the
ordinary: against the definitions in 64 bits of test_tree_gpu."""
import pytest
import torch

from .test_tree_gpu import BF16, attention_oracle, contiguous_cache, make, pack, paged_cache

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
