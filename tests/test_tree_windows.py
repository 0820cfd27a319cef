"""How the work of attention over trees is planned where a window leaves most of the text unseen: read off the scratch that a step wants, without a GPU."""

import pytest
import torch


def scratch(dtype, D, seqs, kv_heads, group, max_nodes, max_kv, window, page_size=16):
    from ferrisinfer_b200.kernels import ops

    ops._lib()
    return ops._tree_attention_scratch(ops._DT[dtype], D, seqs, kv_heads, group, max_nodes, max_kv, page_size, 10 ** 6, 0.1, window, 0)


@pytest.mark.parametrize("dtype, unit", [(torch.bfloat16, 128), (torch.float32, 64)])
@pytest.mark.parametrize("seqs, kv_heads, group, max_nodes", [(1, 1, 1, 1), (8, 2, 2, 16), (2, 2, 7, 9), (1, 4, 4, 64)])
@pytest.mark.parametrize("window", [1, 128, 1000])
def test_only_the_rows_within_the_window_count(dtype, unit, seqs, kv_heads, group, max_nodes, window):
    """(few query rows beside 131,072 cached ones: without the window the bf16 kernel and the number of blocks would be others)"""
    sizes = dtype, 128, seqs, kv_heads, group, max_nodes
    assert scratch(*sizes, 131072, window) == scratch(*sizes, window + max_nodes + unit, 0)
    # (no more blocks than the SMs have room for, which 16 items of 18 tiles take too)
    assert scratch(*sizes, 131072, window) <= scratch(*sizes, 131072, 0)
    assert window > 1 or scratch(*sizes, 131072, window) < scratch(*sizes, 131072, 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_a_window_beyond_the_text_changes_nothing(dtype):
    for window in (5000, 131072, 0x7fffffff):
        assert scratch(dtype, 64, 8, 2, 7, 9, 4200, window) == scratch(dtype, 64, 8, 2, 7, 9, 4200, 0)
