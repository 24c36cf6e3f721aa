"""CPU checks of orders in the kernel sources that no run can be trusted to show."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "torchplusplus_b200" / "csrc"


def kernels_with(word: str) -> list:
    """(file, kernel, body) of every __global__ function that names `word`."""
    found = []
    for path in sorted(CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*|/\*.*?\*/", "", path.read_text(), flags=re.S)
        text = re.sub(r"__launch_bounds__\s*\((?:[^()]|\([^()]*\))*\)", "", text)
        for m in re.finditer(r"__global__[^;{]*?(\w+)\s*\((?:[^;{])*\{", text):
            depth, end = 1, m.end()
            while depth:
                depth += {"{": 1, "}": -1}.get(text[end], 0)
                end += 1
            body = text[m.end():end]
            if re.search(rf"\b{word}\b", body):
                found.append(pytest.param(body, id=f"{path.name}:{m.group(1)}"))
    return found


def test_the_tensor_memory_kernels_are_found():
    assert len(kernels_with("tmem_alloc")) >= 4


@pytest.mark.parametrize("body", kernels_with("tmem_alloc"))
def test_tensor_memory_is_allocated_before_dependents_may_start(body):
    """tcgen05.alloc waits until columns are free, and a dependent kernel that got
    onto the SM first holds its own until this kernel has ended: so a CTA may
    release its dependents (any one thread's pdl_trigger does) only when it has
    its columns, behind a barrier of the CTA."""
    alloc, trigger = body.index("tmem_alloc("), body.index("pdl_trigger(")
    assert alloc < trigger
    assert "__syncthreads()" in body[alloc:trigger]
