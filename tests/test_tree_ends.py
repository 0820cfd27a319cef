"""Rules that the CUDA sources keep about what is still on its way when a block ends, read from their text, without a GPU."""

import re

from test_kernel_sources import block_after, kernels_with


def tree_kernel():
    (_, _, body), = [k for k in kernels_with("tma_load_2d") if k[1] == "tree_attention_tc_kernel"]
    return body


def test_copies_are_awaited_whoever_gave_up():
    """The warp that issued them waits for the last of each stage, also where another warp's wait has run out and its own have not; and behind one that has run out
    itself it issues none, so that no stage has two on their way."""
    body = tree_kernel()
    drained = body.index("148")
    loop = body.rindex("for (", 0, drained)
    assert "issued - ST" in body[loop:drained]
    assert not body[:loop].rstrip().endswith("if (dead)")
    load = body[body.index("auto load = "):]
    load = load[:load.index("tma_load_2d")]
    assert re.search(r"dead = __any_sync\(0xffffffffu, dead\);\s*if \(!dead\) issued = at \+ 1;\s*if \(!dead && lane == 0\) mbar_expect_tx", load)
    assert load.rstrip().rpartition("if (")[2].startswith("!dead && lane <")


def test_products_are_awaited_before_tensor_memory_is_given_back():
    body = tree_kernel()
    last = body.rindex("tcgen05_commit(&ended[g])")
    assert "mbar_wait(&ended[g], 0," in block_after(body, last)
    assert max(body.rindex("tcgen05_mma_bf16("), body.rindex("tcgen05_mma_bf16_ts(")) < last < body.index("tmem_dealloc")
