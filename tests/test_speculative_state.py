"""What a SpeculativeDecoder keeps from one request to the next: the recorded
step and the model's weights that it reads."""
import gc
import weakref

import pytest
import torch
import torch.nn as nn

from torchplusplus_b200.llmops.qwen3 import Qwen3, Qwen3Config
from torchplusplus_b200.llmops.speculative import SpeculativeDecoder


def small_model(device):
    cfg = Qwen3Config(vocab_size=256, context_length=512, embed_dim=256, n_heads=4, n_layers=2,
                      head_dim=64, n_kv_heads=2, hidden_dim=512)
    return Qwen3(cfg, device=device).init_weights(0.05, seed=3)


class FakeGraph:
    """Stands for a recorded step: what it reads is what the model had then."""

    def replay(self):
        pass


@pytest.mark.parametrize("change", ["in_place", "new_parameter", "data"])
def test_what_a_recorded_step_reads_is_kept(change):
    """On the CPU: the storages behind a recorded step outlive a change of the
    weights, and the change is seen."""
    m = small_model(torch.device("cpu"))
    dec = SpeculativeDecoder(m, 1, 32, nodes=4)
    dec._graph, dec._graph_temperature = FakeGraph(), dec.temperature
    dec._graph_weights = [w.detach() for w in dec._weights()]
    blk = m.transformer_blocs[0]
    dec._record()                                   # nothing has changed: no new recording
    old = [weakref.ref(t) for t in (blk.attn._qkv._w, blk.ffn._gu._w)]
    ptrs = {w.data_ptr() for w in dec._graph_weights}
    with torch.no_grad():
        for lin in (blk.attn.Wq, blk.ffn.linear_layerP, blk.ffn.linear_layer2):
            if change == "in_place":
                lin.weight.mul_(1.5)
            elif change == "new_parameter":
                lin.weight = nn.Parameter(lin.weight * 1.5)
            else:
                lin.weight.data = lin.weight.data * 1.5
    now = {w.data_ptr() for w in dec._weights()}
    gc.collect()
    assert all(r() is None for r in old)            # (the concatenations' own owners let go)
    assert {w.data_ptr() for w in dec._graph_weights} == ptrs
    assert len(now - ptrs) == (2 if change == "in_place" else 3)


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_changed_weights_reach_the_next_request(temperature):
    m = small_model(torch.device("cuda", 0))
    ids = torch.arange(30).view(2, 15) % 11
    dec = SpeculativeDecoder(m, 2, 96, nodes=6)
    run = lambda d: d.generate(ids, 30, temperature=temperature, seed=4)
    first = run(dec)
    m.init_weights(0.05, seed=8)                    # in place
    second = run(dec)
    assert second == run(SpeculativeDecoder(m, 2, 96, nodes=6)) and second != first
    with torch.no_grad():                           # other storages
        for blk in m.transformer_blocs:
            blk.ffn.linear_layer2.weight = nn.Parameter(blk.ffn.linear_layer2.weight * -1)
            blk.rms_norm1.weight.data = blk.rms_norm1.weight.data * 0.5
    junk = [torch.full((1 << 18,), float("nan"), device="cuda") for _ in range(64)]
    third = run(dec)
    assert third == run(SpeculativeDecoder(m, 2, 96, nodes=6)) and third != second
    del junk
    m.init_weights(0.05, seed=3)
    for blk in m.transformer_blocs:
        blk.rms_norm1.weight.data.fill_(1.0)
    assert run(dec) == first


@pytest.mark.gpu
def test_recording_leaves_the_lengths_as_they_were(monkeypatch):
    """Work that the caller's stream gets after the recording stream has been
    tied to it (here a pause of some 50 ms) has no part in what is saved."""
    m = small_model(torch.device("cuda", 0))
    dec = SpeculativeDecoder(m, 3, 64, nodes=2)
    dec.ctx.copy_(torch.tensor([3, 9, 0], dtype=torch.int32))
    dec.set_trees([([5], [0])] * 3, [1, 2, 3])
    tie = torch.cuda.Stream.wait_stream

    def tie_then_pause(self, other):
        tie(self, other)
        with torch.cuda.stream(other):
            torch.cuda._sleep(100_000_000)

    torch.cuda.synchronize()
    monkeypatch.setattr(torch.cuda.Stream, "wait_stream", tie_then_pause)
    dec._record()
    torch.cuda.synchronize()
    assert dec.ctx.tolist() == [3, 9, 0]
    dec._replay()
    assert dec.ctx.tolist() == [3 + int(dec.count[0]), 9 + int(dec.count[1]), int(dec.count[2])]


@pytest.mark.gpu
def test_the_norms_own_eps_is_used():
    m = small_model(torch.device("cuda", 0))
    for blk in m.transformer_blocs:
        blk.attn.q_norm.eps = blk.attn.k_norm.eps = 10.0
    ids = torch.arange(24).view(2, 12)
    dec = SpeculativeDecoder(m, 2, 64, nodes=5)
    new = dec.generate(ids, 20)
    ref = SpeculativeDecoder(m, 2, 64, nodes=5)
    n = 12 + 15                                     # rows that both surely hold
    ref.generate(torch.cat([ids, torch.tensor(new)], 1)[:, :n], 1)
    a, b = dec.k[:, :, :, :n].float(), ref.k[:, :, :, :n].float()
    # bf16 rows computed in another order of sums, two layers deep
    assert (a - b).abs().max() <= 2.0 ** -8 * 8 * b.abs().max()


@pytest.mark.gpu
def test_no_new_tokens():
    m = small_model(torch.device("cuda", 0))
    dec = SpeculativeDecoder(m, 2, 64, nodes=5)
    ids = torch.arange(24).view(2, 12)
    assert dec.generate(ids, 0) == [[], []] and dec.steps == 0
    assert [len(n) for n in dec.generate(ids, 1)] == [1, 1]
    with pytest.raises(ValueError):
        dec.generate(ids, -1)
