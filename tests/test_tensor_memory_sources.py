"""The rule of tensor memory for every kernel that takes some, by whatever function: read from the sources' text, without a GPU."""

import os
import re

import pytest

from test_kernel_sources import CSRC, block_after, kernels_with


def takers():
    """Names of the functions that allocate tensor memory, those that call others among them."""
    bodies = {}
    for name in sorted(os.listdir(CSRC)):
        if name.endswith((".cu", ".cuh")):
            with open(os.path.join(CSRC, name)) as f:
                text = re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)
            for m in re.finditer(r"__device__ __forceinline__ \w+ (\w+)\([^)]*\)\s*\{", text):
                bodies[m.group(1)] = block_after(text, m.end())
    found = {f for f, body in bodies.items() if "tcgen05.alloc" in body}
    while more := {f for f, body in bodies.items() if f not in found and any(re.search(rf"\b{g}\(", body) for g in found)}:
        found |= more
    return found


TAKERS = takers()
KERNELS = {k: (file, body) for g in TAKERS for file, k, body in kernels_with(g + "(")}


def test_kernels_that_give_tensor_memory_back_are_those_that_take_it():
    assert TAKERS and KERNELS
    assert set(KERNELS) == {k for _, k, _ in kernels_with("tmem_dealloc")}


@pytest.mark.parametrize("kernel", sorted(KERNELS))
def test_tensor_memory_is_taken_before_dependents_are_let_in(kernel):
    """A dependent launch that is let in first may take an SM's tensor memory and then wait for this one, which waits for it."""
    file, body = KERNELS[kernel]
    taken = min(m.start() for g in TAKERS for m in re.finditer(rf"\b{g}\(", body))
    triggers = [m.start() for m in re.finditer(r"pdl_launch_dependents\(\)", body)]
    assert any(at > taken for at in triggers)
    for at in triggers:
        if at < taken:
            assert "return;" in block_after(body, at), f"{file}: {kernel} lets dependents in before it has its tensor memory"
