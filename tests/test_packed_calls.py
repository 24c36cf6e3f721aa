"""What the packed-prompt wrappers hand to the library, and what they refuse before it, on the
CPU: the library's calls are recorded, none is made."""
import re
from pathlib import Path

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
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
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


class OnGpu(torch.Tensor):
    """A host tensor that says it is on GPU 0 (whatever is made from it too)."""
    is_cuda = property(lambda self: True)

    def get_device(self):
        return 0


def on_gpu(t):
    return t.as_subclass(OnGpu)


def within(t, address, stride, N, E):
    """Whether rows of E elements lie inside t's memory."""
    lo = t.untyped_storage().data_ptr()
    end = address + ((N - 1) * stride + E) * t.element_size()
    return lo <= address and end <= lo + t.untyped_storage().nbytes()


@pytest.mark.parametrize("step", [8, 24, 56])
@pytest.mark.parametrize("which", ["x", "weight"])
def test_linear_logprobs_of_rows_that_overlap(calls, which, step):
    """Rows that share memory (a row stride below their length) are copied apart."""
    N_, V, E = 5, 7, 64
    rows = dict(x=N_, weight=V)
    got = dict(x=on_gpu(torch.zeros(N_, E, dtype=BF16)), weight=on_gpu(torch.zeros(V, E, dtype=BF16)))
    room = on_gpu(torch.zeros((rows[which] - 1) * step + E, dtype=BF16))
    got[which] = room.as_strided((rows[which], E), (step, 1))
    ops.linear_logprobs(got["x"], got["weight"], on_gpu(torch.zeros(N_, dtype=torch.int64)))
    (_, args), = calls
    address, stride = args[0 if which == "x" else 2], args[1 if which == "x" else 3]
    assert stride >= E
    # (a copy's memory has been freed by now; the operand's own must not be read that far)
    assert address != room.data_ptr() or within(room, address, stride, rows[which], E)


def pitched(rows, *shape, dtype=BF16):
    """Rows of `shape` at a pitch that is no multiple of 16 bytes."""
    n = torch.Size(shape).numel()
    return on_gpu(torch.zeros(rows, n + 5, dtype=dtype))[:, :n].view(rows, *shape)


def test_the_stride_of_a_single_row_does_not_matter(calls):
    """A tensor of one row may lie in memory of any pitch: no stride that the library would
    refuse (a multiple of 8 elements) gets there."""
    cu = on_gpu(torch.tensor([0, 1], dtype=torch.int32))
    one = on_gpu(torch.zeros(1, dtype=torch.int64))
    ops.linear_logprobs(pitched(3, 64)[:1], pitched(3, 64)[:1], one)
    ops.attention_packed(pitched(2, 4, 64)[:1], pitched(2, 2, 64)[:1], pitched(2, 2, 64)[:1], cu,
                         out=pitched(2, 4, 64)[:1])
    table = on_gpu(torch.ones(8, 64))
    for kc, vc in ((None, None), (pitched(2, 2, 8, 64)[:1], pitched(2, 2, 8, 64)[:1])):
        ops.qk_norm_rope_packed(pitched(2, 8 * 64)[:1], None, None, 1e-6, table, table, cu, 4, 2, kc, vc)
    strides = {"tpp_linear_logprobs": [1, 3], "tpp_attention_packed": [1, 2, 4, 5, 7, 8, 12, 13],
               "tpp_qk_norm_rope_packed": [1, 7, 16, 17, 18]}
    assert len(calls) == 4
    for name, args in calls:
        assert not [args[i] for i in strides[name] if args[i] % 8], name


class TwoGpus:
    """A library for two devices whose workspaces differ in size."""
    need = {0: 1024, 1: 4096}

    def __init__(self):
        self.current, self.called = 0, []

    def tpp_linear_logprobs_workspace(self, N_, V, E):
        return self.need[self.current]

    def tpp_linear_logprobs(self, *args):
        nbytes = args[12]
        self.called.append((self.current, nbytes))
        return 0 if nbytes >= self.need[self.current] else 7

    def tpp_last_error(self):
        return b"workspace missing or too small"


@pytest.fixture
def two_gpus(monkeypatch):
    gpus = TwoGpus()

    class device:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            self.old, gpus.current = gpus.current, self.dev

        def __exit__(self, *_):
            gpus.current = self.old
    monkeypatch.setattr(N, "_lib", gpus)
    monkeypatch.setattr(N, "stream_of", lambda t: 0)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: gpus.current, raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    return gpus


class OnGpu1(OnGpu):
    def get_device(self):
        return 1


def test_linear_logprobs_workspace_is_of_the_operands_device(two_gpus):
    """Its size goes by the SMs of the device that the call runs on, not of the current one."""
    x, w = (torch.zeros(5, 64, dtype=BF16).as_subclass(OnGpu1) for _ in range(2))
    ops.linear_logprobs(x, w, torch.zeros(5, dtype=torch.int64).as_subclass(OnGpu1))
    assert two_gpus.called == [(1, 4096)] and two_gpus.current == 0
    assert ops.linear_logprobs_workspace_bytes(5, 5, 64) == 1024
    assert ops.linear_logprobs_workspace_bytes(5, 5, 64, torch.device("cuda", 1)) == 4096


def wait_codes(path):
    """The codes that a kernel source's bounded waits set when they run out."""
    text = re.sub(r"//[^\n]*", "", path.read_text())
    return [int(c) for c in re.findall(r"\w*wait\w*\([^;]*?, *(\d+)\)[;) ]", text)
            + re.findall(r"expired\w*\([^;]*?, *(\d+)\)", text)]


@pytest.mark.parametrize("name", ["packed_attn.cu", "linear_logprobs.cu"])
def test_a_wait_that_ran_out_can_be_told_from_the_others(name):
    csrc = Path(ops.__file__).parent / "csrc"
    mine = wait_codes(csrc / name)
    assert len(mine) >= 4 and len(set(mine)) == len(mine)
    others = {c for p in csrc.glob("*.cu") if p.name != name for c in wait_codes(p)}
    assert not others & set(mine)
