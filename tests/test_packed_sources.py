"""The prompts' kernels over the packed cache keep the rule of tensor memory: it is allocated before dependent launches are let in."""

import re

from test_kernel_sources import block_after, kernels_with


def test_tensor_memory_is_allocated_before_dependents_are_let_in():
    found = kernels_with("tensor_memory_begin")
    assert {k for _, k, _ in found} == {"packed_prefill_kernel", "packed_prefill_weights_kernel"}
    for file, kernel, body in found:
        allocated = body.index("tensor_memory_begin")
        triggers = [m.start() for m in re.finditer(r"pdl_launch_dependents\(\)", body)]
        assert any(at > allocated for at in triggers)
        for at in triggers:
            if at < allocated:
                assert "return;" in block_after(body, at), f"{file}: {kernel} lets dependents in before it has its tensor memory"


def test_the_kernels_that_share_tensor_memory_wait_within_limits():
    """Their waits are those with a limit; a wait that runs out leaves nobody at a barrier of some of the warps."""
    for _, kernel, body in kernels_with("tensor_memory_begin"):
        assert "try_wait" not in body and "mbar_wait(" in body
        loops = [m.start() for m in re.finditer(r"\bbreak;", body)]
        assert not loops, f"{kernel}: a loop that ends early could leave others at a named barrier"
