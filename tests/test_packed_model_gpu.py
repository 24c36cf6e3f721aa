"""Packed prompts through the model, the engine and the attention modules, against the fp32
oracle model and against the same prompts one at a time."""
import pytest
import torch

from oracle import model as OM
from torchplusplus_b200.llmops.qwen3 import Qwen3, Qwen3Config

pytestmark = pytest.mark.gpu
DEV = "cuda"
LENS = [40, 1, 2, 129, 65]


def make(dtype=torch.bfloat16, head_dim=64, seed=0):
    cfg = Qwen3Config(vocab_size=1000, context_length=512, embed_dim=256, n_heads=4, n_layers=2,
                      head_dim=head_dim, n_kv_heads=2, hidden_dim=512, dtype=dtype)
    return Qwen3(cfg).to(DEV).init_weights(std=0.05, seed=seed)


def prompts(lens=LENS, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 1000, (n,), generator=g) for n in lens]


def oracle_logits(m, ids):
    return OM.forward(m.state_dict(), m.cfg, ids[None])[0]


def bound(ref):
    """How far a logit of the 16-bit model may be from the fp32 oracle's (the model tests' bound)."""
    return 2e-2 * max(1.0, ref.abs().max().item())


@pytest.mark.parametrize("dtype,head_dim", [(torch.bfloat16, 64), (torch.float16, 128)])
@pytest.mark.parametrize("top", [None, 0, 5])
def test_scores_match_the_oracle_model(dtype, head_dim, top):
    m = make(dtype, head_dim)
    ps = prompts()
    got = m.score(ps, top=top)
    assert [len(s.logprobs) for s in got] == [max(0, n - 1) for n in LENS]
    for p, s in zip(ps, got):
        if len(p) < 2:
            continue
        ref = oracle_logits(m, p)
        l = torch.log_softmax(ref.double(), 1)[:-1]
        tol = 2 * bound(ref)
        assert (s.logprobs.cpu() - l.gather(1, p[1:, None])[:, 0]).abs().max() <= tol
        # d entropy / d logit sums to at most twice the entropy
        assert (s.entropy.cpu() + (l.exp() * l).sum(1)).abs().max() <= 2 * 6.91 * bound(ref)
        if top:
            best = l.topk(top).values
            assert (s.top_logprobs.cpu() - best).abs().max() <= tol
            assert s.top_tokens.shape == (len(p) - 1, top) and s.ranks.min() >= 1
            at = l.gather(1, s.top_tokens.cpu())
            assert (s.top_logprobs.cpu() - at).abs().max() <= tol


def test_scores_do_not_depend_on_the_company():
    """A prompt's scores packed with others and alone."""
    m = make()
    ps = prompts()
    a = m.score(ps)
    for p, s in zip(ps, a):
        b = m.score([p])[0]
        tol = 2 * bound(oracle_logits(m, p))
        if len(p) > 1:
            assert (s.logprobs - b.logprobs).abs().max() <= tol


def test_scores_at_a_temperature_and_of_nothing():
    m = make()
    p = prompts([30])[0]
    l = torch.log_softmax(oracle_logits(m, p).double() / 0.5, 1)[:-1].gather(1, p[1:, None])[:, 0]
    got = m.score([p], temperature=0.5)[0]
    assert (got.logprobs.cpu() - l).abs().max() <= 4 * bound(oracle_logits(m, p))
    assert [len(s.logprobs) for s in m.score([p[:0], p[:1]])] == [0, 0]
    e = m.score([p[:0]], top=3)[0]
    assert e.top_tokens.shape == (0, 3)
    with pytest.raises(ValueError):
        m.score([])
    with pytest.raises(ValueError):
        m.score([torch.zeros(600, dtype=torch.int64)])
    with pytest.raises(ValueError):
        m.score([p[None]])


@pytest.mark.parametrize("batch", [1, 5])
def test_generate_from_prompts_of_different_lengths(batch):
    """Each greedy pick is an argmax of the oracle's logits up to the model's bound, through
    packed prefill, the caches that it fills and the decode steps on them."""
    m = make()
    ps = prompts(LENS[:batch])
    out = m.generate(ps, max_new_token=12, sampling_strategy="greedy")
    assert [len(o) for o in out] == [len(p) + 12 for p in ps]
    for p, o in zip(ps, out):
        o = o.cpu()
        assert torch.equal(o[:len(p)], p)
        ref = oracle_logits(m, o)
        pick = ref[len(p) - 1:-1]
        assert (pick.amax(1) - pick.gather(1, o[len(p):, None])[:, 0]).max() <= 2 * bound(ref)


def test_packed_prefill_matches_a_batch_of_one_length():
    m = make()
    ids = torch.stack(prompts([50, 50, 50]))
    a = m.generate(ids, max_new_token=8, sampling_strategy="greedy").cpu()
    eng = m.engine(3, 58)
    la = eng.logits.float().clone()
    b = m.generate(list(ids), max_new_token=8, sampling_strategy="greedy")
    assert torch.equal(torch.stack(b).cpu(), a)
    assert (eng.logits.float() - la).abs().max() <= 2 * bound(la)


@pytest.mark.parametrize("batch", [1, 3])
@pytest.mark.parametrize("sampled", [False, True])
def test_engine_scores_of_the_tokens_chosen(batch, sampled):
    from torchplusplus_b200 import ops
    m = make()
    ps = prompts([20, 33, 7][:batch])
    eng = m.engine(batch, 64)
    if sampled:
        eng.set_sampling(temperature=0.8, top_k=20, seed=5)
    eng.set_logprobs(3)
    out = eng.generate(ps, 10)
    lp, ent, rank, tlp, tid = eng.scores
    for b, (p, o) in enumerate(zip(ps, out)):
        n = len(p)
        assert (lp[b, :n] == 0).all() and (rank[b, :n] == 0).all() and (lp[b, n + 10:] == 0).all()
        assert (rank[b, n:n + 10] >= 1).all() and (sampled or (rank[b, n:n + 10] == 1).all())
        want = m.score([o])[0]
        tol = 2 * bound(oracle_logits(m, o.cpu()))
        assert (lp[b, n:n + 10] - want.logprobs[n - 1:]).abs().max() <= tol
        assert (tid[b, n:n + 10] < 1000).all() and (tlp[b, n:n + 10].diff(dim=1) <= 0).all()
        if not sampled:
            assert torch.equal(tid[b, n:n + 10, 0], o[n:])
    # the last step's, from the logits that it left
    now = ops.token_logprobs(eng.logits, eng.tokens, top=3)
    at = eng.positions.long()
    for room, t in zip(eng.scores, now):
        assert torch.equal(room[torch.arange(batch, device=DEV), at], t)
    # a second request, without them and with others
    eng.set_logprobs(None)
    again = eng.generate(ps, 10)
    assert eng.scores is None and all(torch.equal(x, y) for x, y in zip(out, again))
    eng.set_logprobs(0)
    eng.generate(ps, 10)
    assert torch.equal(eng.scores[0], lp) and eng.scores[3].shape[-1] == 0
    with pytest.raises(ValueError):
        eng.set_logprobs(33)


def test_engine_refuses_what_does_not_fit():
    m = make()
    eng = m.engine(2, 32)
    for bad in (prompts([3]), prompts([3, 0]), prompts([3, 32]), prompts([3, 4, 5])):
        with pytest.raises(ValueError):
            eng.prefill(bad)
    with pytest.raises(ValueError):
        m.generate(prompts([3, 4]), 4, sampling_strategy="top_k")


def test_sliding_window_module_packed():
    from torchplusplus_b200.attention.swa import SlidingWindowAttention
    from torchplusplus_b200.dlops.rope import compute_rope_params
    torch.manual_seed(0)
    a = SlidingWindowAttention(33, 256, 4, dtype=torch.bfloat16, n_kv_heads=2).to(DEV)
    cos, sin = compute_rope_params(64, 1e6, 256, device=DEV)
    lens = [100, 1, 150]
    x = torch.randn(sum(lens), 256, device=DEV).to(torch.bfloat16)
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(DEV)
    with torch.inference_mode():
        got = a.forward_packed(x, cos, sin, cu).float()
        s = 0
        for n in lens:
            want = a(x[None, s:s + n], cos, sin)[0].float()
            # both round the probabilities, the attention's and the projection's outputs to bf16
            assert (got[s:s + n] - want).abs().max() <= 2e-2 * max(1.0, want.abs().max().item())
            s += n


def test_generate_refuses_prompts_of_no_tokens():
    m = make()
    for bad in ([], [torch.tensor([3, 4]), torch.tensor([], dtype=torch.int64)]):
        with pytest.raises(ValueError):
            m.generate(bad, max_new_token=4, sampling_strategy="greedy")
