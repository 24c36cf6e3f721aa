"""CPU checks of the packed-prompt operators: arguments that the C-ABI and the wrappers refuse
before any launch, workspace sizes, packing."""
import pytest
import torch

from torchplusplus_b200 import _native as N
from torchplusplus_b200 import ops
from torchplusplus_b200.llmops import pack

A = 4096  # an aligned address that is never read


def attention(q=A, sn=256, sh=128, B=1, rows=10, Hq=2, Hkv=2, D=128, scale=1.0, dtype=1, o=A):
    N.call("tpp_attention_packed", q, sn, sh, A, 256, 128, A, 256, 128, A, B, o, 256, 128, rows, Hq,
           Hkv, D, 1, -1, scale, dtype, None)


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), 1), (dict(Hq=3), 1), (dict(Hkv=0), 1), (dict(rows=-1), 1), (dict(D=96), 6),
    (dict(Hq=258), 6), (dict(sn=257), 3), (dict(q=A + 2), 3), (dict(scale=float("nan")), 1),
    (dict(o=A + 8), 3), (dict(rows=1 << 31), 1), (dict(rows=1 << 29, Hq=1 << 12, Hkv=1 << 12), 1)])
def test_attention_refuses(kw, status):
    with pytest.raises(N.TppError) as e:
        attention(**kw)
    assert e.value.status == status


def test_nothing_to_do_is_no_error():
    attention(rows=0)
    attention(B=0)
    N.call("tpp_token_logprobs", None, 0, 0, 5, None, 1.0, 0, None, None, None, None, None, 1, None)
    N.call("tpp_linear_logprobs", None, 0, None, 0, None, 0, 5, 8, 1.0, None, None, None, 0, 1, None)


def logprobs(x=A, ld=100, rows=3, V=100, t=1.0, top=0, out=A, tops=A, dtype=1):
    N.call("tpp_token_logprobs", x, ld, rows, V, A, t, top, out, A, A, tops, tops, dtype, None)


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), 1), (dict(out=None), 1), (dict(V=0), 1), (dict(ld=99), 1), (dict(t=0.0), 1),
    (dict(t=-1.0), 1), (dict(t=float("nan")), 1), (dict(t=float("inf")), 1), (dict(top=33), 1),
    (dict(top=-1), 1), (dict(V=4, ld=4, top=5), 1), (dict(top=2, tops=None), 1), (dict(dtype=7), 2),
    (dict(V=1 << 31, ld=1 << 31), 1)])
def test_token_logprobs_refuses(kw, status):
    with pytest.raises(N.TppError) as e:
        logprobs(**kw)
    assert e.value.status == status


def head(x=A, ldx=64, ldw=64, rows=3, V=100, E=64, t=1.0, ws=A, nbytes=1 << 30, dtype=1):
    N.call("tpp_linear_logprobs", x, ldx, A, ldw, A, rows, V, E, t, A, A, ws, nbytes, dtype, None)


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), 1), (dict(E=60), 3), (dict(ldx=72 + 4), 3), (dict(ldx=56), 1), (dict(x=A + 2), 3),
    (dict(t=0.0), 1), (dict(ws=None), 7), (dict(nbytes=16), 7), (dict(V=0), 1)])
def test_linear_logprobs_refuses(kw, status):
    with pytest.raises(N.TppError) as e:
        head(**kw)
    assert e.value.status == status


@pytest.mark.parametrize("rows,V", [(1, 1), (128, 256), (129, 151936), (4096, 32003)])
def test_linear_logprobs_workspace_holds_a_tile_row_of_statistics(rows, V):
    need = ops.linear_logprobs_workspace_bytes(rows, V, 64)
    up = (rows + 127) // 128 * 128
    # three numbers a row and tile of 128 to 256 vocabulary rows, and the token's logit
    assert 4 * up * (3 * -(-V // 256) + 1) <= need <= 4 * up * (3 * -(-V // 128) + 1)
    assert ops.linear_logprobs_workspace_bytes(0, V, 64) == 0


def rope(qkv=A, sn=1024, B=1, rows=5, Hq=4, Hkv=2, D=128, kc=None, vc=None, cs=2, qn=None):
    N.call("tpp_qk_norm_rope_packed", qkv, sn, qn, None, 1e-6, A, A, D, 10, cs, A, B, A, A, kc, vc, 0,
           0, 0, 0, 0, None, 0, rows, Hq, Hkv, D, 1, None)


@pytest.mark.parametrize("kw,status", [
    (dict(qkv=None), 1), (dict(kc=A), 1), (dict(Hkv=0), 1), (dict(D=48), 6), (dict(sn=1025), 3),
    (dict(cs=9), 2), (dict(qn=A + 2), 3), (dict(rows=1 << 30, Hq=8), 1)])
def test_rope_refuses(kw, status):
    with pytest.raises(N.TppError) as e:
        rope(**kw)
    assert e.value.status == status


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError):
        ops.attention_packed(x, x, x, cu)
    with pytest.raises(RuntimeError):
        ops.token_logprobs(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError):
        ops.linear_logprobs(x[0], x[1], torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError):
        ops.qk_norm_rope_packed(x.view(4, -1), None, None, 1e-6, torch.ones(4, 32), torch.ones(4, 32),
                                cu, 2, 1)


def test_pack():
    ids, cu, lens = pack([torch.tensor([5, 6]), torch.tensor([], dtype=torch.int64),
                          torch.tensor([7], dtype=torch.int32)], "cpu")
    assert ids.tolist() == [5, 6, 7] and ids.dtype == torch.int64
    assert cu.tolist() == [0, 2, 2, 3] and cu.dtype == torch.int32 and lens == [2, 0, 1]
    for bad in ([], [torch.zeros(2, 2)], [torch.zeros(3)]):
        with pytest.raises(ValueError):
            pack(bad, "cpu")
