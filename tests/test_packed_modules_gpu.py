"""forward_packed of the attention modules and the model: what does not fit is refused, as
forward refuses it."""
import pytest
import torch

from torchplusplus_b200.attention.gqa import GroupedQueryAttention
from torchplusplus_b200.attention.swa import SlidingWindowAttention
from torchplusplus_b200.dlops.rope import compute_rope_params
from torchplusplus_b200.llmops.kvcache import KVCache

from .test_packed_model_gpu import make, prompts

pytestmark = pytest.mark.gpu
DEV, BF16 = "cuda", torch.bfloat16


def module(kind):
    torch.manual_seed(0)
    if kind == "gqa":
        return GroupedQueryAttention(256, 4, 2, dtype=BF16).to(DEV)
    return SlidingWindowAttention(33, 256, 4, dtype=BF16, n_kv_heads=2).to(DEV)


def packed(lens, tail=0):
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    return torch.randn(sum(lens) + tail, 256, generator=g, device=DEV).to(BF16), cu


def cache(batch, rows):
    return KVCache(rows, 2, 64, BF16, torch.device(DEV), batch_size=batch)


@pytest.mark.parametrize("kind", ["gqa", "swa"])
@torch.inference_mode()
def test_prompts_longer_than_the_cache_or_the_tables(kind):
    a = module(kind)
    cos, sin = compute_rope_params(64, 1e6, 100, device=DEV)
    x, cu = packed([60, 3, 90])
    for kw in (dict(), dict(max_seqlen=90)):
        with pytest.raises(ValueError, match="KV cache overflow"):
            a.forward_packed(x, cos, sin, cu, cache(3, 89), **kw)
        with pytest.raises(ValueError, match="rotary table"):
            a.forward_packed(x, cos[:89], sin[:89], cu, cache(3, 90), **kw)
        with pytest.raises(ValueError, match="rotary table"):
            a.forward_packed(x, cos[:89], sin[:89], cu, **kw)
        # all rows together are more than the cache and the tables hold, each prompt is not
        kv = cache(3, 90)
        got = a.forward_packed(x, cos[:90], sin[:90], cu, kv, **kw)
        assert torch.equal(got, a.forward_packed(x, cos, sin, cu)) and kv.k_cache[2, :, 89].any()


@torch.inference_mode()
def test_rows_of_no_prompt_do_not_count():
    a = module("gqa")
    cos, sin = compute_rope_params(64, 1e6, 40, device=DEV)
    x, cu = packed([40, 3], tail=50)
    got = a.forward_packed(x, cos, sin, cu, cache(2, 40))
    assert torch.equal(got[:43], a.forward_packed(x[:43], cos, sin, cu))
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert a.forward_packed(x, cos, sin, none).shape == x.shape


@torch.inference_mode()
def test_recorded_calls_say_their_longest_prompt():
    """A call that is being recorded cannot look at the lengths on the device."""
    a = module("gqa")
    cos, sin = compute_rope_params(64, 1e6, 60, device=DEV)
    x, cu = packed([60, 3])
    want = a.forward_packed(x, cos, sin, cu)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        with pytest.raises(ValueError, match="max_seqlen"):
            a.forward_packed(x, cos, sin, cu)
        got = a.forward_packed(x, cos, sin, cu, max_seqlen=60)
    g.replay()
    assert torch.equal(got, want)


@pytest.mark.parametrize("kind", ["gqa", "swa"])
@torch.inference_mode()
def test_without_rotary_tables(kind):
    a = module(kind)
    lens = [100, 1, 70]
    x, cu = packed(lens)
    got = a.forward_packed(x, None, None, cu).float()
    s = 0
    for n in lens:
        want = a(x[None, s:s + n], None, None)[0].float()
        # both round the probabilities, the attention's and the projection's outputs to bf16
        assert (got[s:s + n] - want).abs().max() <= 2e-2 * max(1.0, want.abs().max().item())
        s += n


@torch.inference_mode()
def test_model_prompts_longer_than_its_tables_or_caches():
    m = make()  # (a context of 512)
    ids = torch.cat(prompts([513, 2])).to(DEV)
    cu = torch.tensor([0, 513, 515], dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="rotary table"):
        m.forward_packed(ids, cu)
    ids, cu = ids[1:], (cu - 1).clamp_min(0)
    whole = m.forward_packed(ids, cu)
    assert torch.equal(m.forward_packed(ids, cu, max_seqlen=512), whole)
    caches = [KVCache(511, 2, 64, BF16, torch.device(DEV), batch_size=2) for _ in range(2)]
    with pytest.raises(ValueError, match="KV cache overflow"):
        m.forward_packed(ids, cu, caches)


def test_scores_asked_for_in_inference_mode():
    """What set_logprobs allocates there is written by steps outside it too."""
    m = make()
    want = None
    for inside in (False, True):
        eng = m.engine(2, 64)
        with torch.inference_mode(inside):
            eng.set_logprobs(None)
            eng.set_logprobs(2)
        eng.set_greedy()
        eng.prefill(prompts([20, 7]))
        eng.decode(3)
        eng.step_eager()
        got = [s.clone() for s in eng.scores]
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert (got[2][0, 20:25] == 1).all() and (got[2][1, 7:12] == 1).all()


@pytest.mark.parametrize("batch", [2, 5])
def test_scores_of_a_batch_in_lanes(batch):
    """Each lane scores its own sequences, side by side in the graph."""
    from torchplusplus_b200.llmops.engine import DecodeEngine
    m = make()
    ps = prompts([20, 33, 7, 50, 1][:batch])
    for lanes in (1, 2):
        eng = DecodeEngine(m, batch, 96, lanes=lanes)
        eng.set_logprobs(4)
        out = eng.generate(ps, 12)
        for b, (p, o) in enumerate(zip(ps, out)):
            n = len(p)
            now = torch.arange(n, n + 12, device=DEV)
            assert torch.equal(eng.scores[4][b, now, 0], o[n:]) and (eng.scores[2][b, now] == 1).all()
            assert (eng.scores[0][b, now] < 0).all() and (eng.scores[0][b, n + 12:] == 0).all()
