"""Speculative decoding with draft trees: the tree helpers (CPU) and the decoder
against the model itself (GPU)."""
import pytest
import torch

from torchplusplus_b200.llmops.speculative import lookup_draft, tree_mask


def test_tree_mask_and_depth():
    #      0
    #    1   2
    #   3    4 5
    mask, depth = tree_mask(torch.tensor([-1, 0, 0, 1, 2, 2]))
    assert depth.tolist() == [0, 1, 1, 2, 2, 2]
    assert mask[:, 0].tolist() == [0b1, 0b11, 0b101, 0b1011, 0b10101, 0b100101]
    chain = torch.arange(-1, 69)
    mask, depth = tree_mask(torch.stack([chain, chain.clamp_max(0)]))
    assert mask.shape == (2, 70, 2) and depth[0].tolist() == list(range(70))
    assert mask[0, 69].tolist() == [-1, 0b111111] and mask[1, 69].tolist() == [1, 1 << 5]
    with pytest.raises(ValueError):
        tree_mask(torch.tensor([-1, 1]))


def test_lookup_draft_merges_continuations():
    h = [1, 2, 3, 9, 1, 2, 4, 8, 1, 2]
    tokens, parents = lookup_draft(h, 7)
    # the last occurrence of (1, 2) goes on with 4 8 1 2, the one before with 3 9 1 ..
    assert tokens == [4, 8, 1, 2, 3, 9] and parents == [0, 1, 2, 3, 0, 5]
    assert lookup_draft([5], 4) == ([], []) and lookup_draft([1, 2, 3], 4) == ([], [])
    t, p = lookup_draft([7, 7, 7, 7], 3)
    assert len(t) <= 2 and all(a <= i for i, a in enumerate(p))


@pytest.fixture(scope="module")
def model():
    from torchplusplus_b200.llmops.qwen3 import Qwen3, Qwen3Config
    cfg = Qwen3Config(vocab_size=256, context_length=512, embed_dim=256, n_heads=4, n_layers=3,
                      head_dim=64, n_kv_heads=2, hidden_dim=512)
    return Qwen3(cfg, device=torch.device("cuda", 0)).init_weights(0.05, seed=3)


def greedy_regret(model, ids, new):
    """How far each emitted token's logit is below the largest, at most, and the
    logits' size, from one forward pass over the whole sequence."""
    full = torch.cat([ids, torch.tensor(new)], 1).cuda()
    with torch.inference_mode():
        logits = model.forward_impl(full[:, :-1]).float()[:, ids.shape[1] - 1:]
    took = logits.gather(2, full[:, ids.shape[1]:, None])[..., 0]
    return float((logits.amax(-1) - took).max()), float(logits.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("nodes", [1, 6, 20, 70])
def test_greedy_emits_the_models_argmax(model, nodes):
    from torchplusplus_b200.llmops.speculative import SpeculativeDecoder
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(0, 256, (3, 20), generator=g)
    ids[1, 10:] = ids[1, :10]                       # something to look up
    dec = SpeculativeDecoder(model, 3, 160, nodes=nodes)
    new = dec.generate(ids, 60)
    assert [len(n) for n in new] == [60, 60, 60]
    # the model's tolerance for bf16 logits against another order of the sums
    regret, size = greedy_regret(model, ids, new)
    assert regret <= 2 * 2e-2 * max(1.0, size)
    assert dec.steps <= 59
    # the same again: nothing is left over from the request before
    assert dec.generate(ids, 60) == new


@pytest.mark.gpu
@pytest.mark.parametrize("nodes", [2, 7, 65])
def test_right_drafts_are_accepted_in_one_step(model, nodes):
    """Drafts of the model's own continuation, among wrong siblings, are taken as
    far as the model's choice is clear of its tolerance."""
    from torchplusplus_b200.llmops.speculative import SpeculativeDecoder
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(0, 256, (1, 16), generator=g)
    new = SpeculativeDecoder(model, 1, 128, nodes=1).generate(ids, 40)
    full = torch.cat([ids, torch.tensor(new)], 1).cuda()
    with torch.inference_mode():
        top = model.forward_impl(full[:, :-1]).float()[0, 15:].topk(2, -1).values
    gap = (top[:, 0] - top[:, 1]).cpu()
    clear = int((gap > 2 * 2e-2 * max(1.0, float(top.abs().max()))).long().cumprod(0).sum())
    take = min(clear - 1, (nodes - 1) // 2 if nodes > 2 else 1)   # drafted tokens that must pass

    def draft(history, n):
        at = len(history) - 16
        tokens, parents, cur = [], [], 0
        for t in new[0][at:at + take]:
            if nodes > 2:                       # a wrong sibling first
                tokens.append((t + 1) % 256)
                parents.append(cur)
            tokens.append(t)
            parents.append(cur)
            cur = len(tokens)
        return tokens, parents

    if take < 1:
        pytest.skip("the model's first choice is not clear")
    dec = SpeculativeDecoder(model, 1, 128, nodes=nodes, draft=draft)
    assert dec.generate(ids, take + 2)[0][:take + 1] == new[0][:take + 1] and dec.steps == 1


@pytest.mark.gpu
def test_cache_holds_what_a_prefill_would_write(model):
    from torchplusplus_b200.llmops.speculative import SpeculativeDecoder
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 256, (2, 12), generator=g)
    dec = SpeculativeDecoder(model, 2, 128, nodes=9)
    new = dec.generate(ids, 40)
    ref = SpeculativeDecoder(model, 2, 128, nodes=9)
    n = 12 + 30                                     # rows that both surely hold
    ref.generate(torch.cat([ids, torch.tensor(new)], 1)[:, :n], 1)
    for a, b in ((dec.k, ref.k), (dec.v, ref.v)):
        a, b = a[:, :, :, :n].float(), b[:, :, :, :n].float()
        # bf16 rows computed in another order of sums, three layers deep
        assert (a - b).abs().max() <= 2.0 ** -8 * 8 * b.abs().max()


@pytest.mark.gpu
def test_sampling_is_seeded_and_stops_at_eos(model):
    from torchplusplus_b200.llmops.speculative import SpeculativeDecoder
    ids = torch.arange(24).view(2, 12)
    dec = SpeculativeDecoder(model, 2, 96, nodes=8)
    a = dec.generate(ids, 40, temperature=0.8, seed=5)
    assert a == dec.generate(ids, 40, temperature=0.8, seed=5)
    assert a != dec.generate(ids, 40, temperature=0.8, seed=6)
    eos = a[0][7]
    b = dec.generate(ids, 40, temperature=0.8, seed=5, eos_token_id=eos)
    assert b[0][-1] == eos and len(b[0]) <= 8 and b[0] == a[0][:len(b[0])]


@pytest.mark.gpu
def test_refusals(model):
    from torchplusplus_b200.llmops.speculative import SpeculativeDecoder
    with pytest.raises(ValueError):
        SpeculativeDecoder(model, 1, 64, nodes=257)
    with pytest.raises(ValueError):
        SpeculativeDecoder(model, 1, 512, nodes=8)       # the rotary table ends there
    dec = SpeculativeDecoder(model, 1, 32, nodes=4)
    with pytest.raises(ValueError):
        dec.generate(torch.zeros(1, 20, dtype=torch.int64), 13)
    with pytest.raises(ValueError):
        dec.generate(torch.zeros(2, 4, dtype=torch.int64), 3)
