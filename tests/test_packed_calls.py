"""What the packed-prompt wrappers hand to the library, and what they refuse before it, on the
CPU: the library's calls are recorded, none is made."""
import pytest
import torch

from torchplusplus_b200 import _native as N
from torchplusplus_b200 import ops

BF16 = torch.bfloat16


@pytest.fixture
def calls(monkeypatch):
    """The calls that would have been made: (name, arguments)."""
    made = []
    monkeypatch.setattr(N, "call_on", lambda t, name, *args: made.append((name, args)))
    monkeypatch.setattr(N, "stream_of", lambda t: 0)
    return made


def cpu_calls():
    x = torch.zeros(4, 2, 64, dtype=BF16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    one = torch.ones(4, 32)
    tokens = torch.zeros(2, dtype=torch.int64)
    return {
        "attention_packed": lambda: ops.attention_packed(x, x, x, cu),
        "qk_norm_rope_packed": lambda: ops.qk_norm_rope_packed(
            x.view(4, -1), None, None, 1e-6, one, one, cu, 2, 1),
        "token_logprobs": lambda: ops.token_logprobs(torch.zeros(2, 5), tokens),
        "token_logprobs of no rows": lambda: ops.token_logprobs(torch.zeros(0, 5), tokens[:0]),
        "linear_logprobs": lambda: ops.linear_logprobs(x[0], x[1], tokens)}


@pytest.mark.parametrize("name", list(cpu_calls()))
def test_cpu_tensors_never_reach_the_library(calls, name):
    with pytest.raises(RuntimeError, match="need CUDA tensors"):
        cpu_calls()[name]()
    assert calls == []
