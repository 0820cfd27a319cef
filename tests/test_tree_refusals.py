"""Memory that is shared, as the C entries of the operators over drafted tokens refuse it; every call here is refused, so nothing runs."""

import pytest
import torch

from test_tree_sources import attention_arguments, refusal, verification_arguments

MB = 1 << 20


def attention(dtype, q, out, k=64 * MB, v=128 * MB, **more):
    from ferrisinfer_b200.kernels import ops

    return attention_arguments(dtype=ops._DT[dtype], q=q, out=out, k=k, v=v, **more)


@pytest.mark.parametrize("dtype, item", [(torch.bfloat16, 2), (torch.float32, 4)], ids=["bf16", "fp32"])
@pytest.mark.parametrize("q, out, ldq, ldo", [
    (0, 0, 256, 256), (0, 0, 768, 768), (0, 2, 768, 768), (4, 0, 768, 768), (0, 255, 768, 768), (255, 0, 768, 768),
    (0, 700, 768, 768),                                     # the end of a row and the beginning of the next one
    (0, 768, 768, 768), (0, 8, 768, 256), (8, 0, 768, 256), (0, 0, 0, 256), (0, 0, 0, 0),
])
def test_an_attention_into_its_queries_is_refused(dtype, item, q, out, ldq, ldo):
    """(256 columns; where they begin and how far rows are apart in elements)"""
    assert "apart from the queries" in refusal("ferris_tree_attention", attention(dtype, MB + q * item, MB + out * item, ldq=ldq, ldo=ldo))


@pytest.mark.parametrize("dtype, item", [(torch.bfloat16, 2), (torch.float32, 4)], ids=["bf16", "fp32"])
@pytest.mark.parametrize("which", ["k", "v"])
def test_an_attention_into_its_cache_is_refused(dtype, item, which):
    cache, out_bytes = 4 * 2 * 16 * 64 * item, 3 * 256 * item
    for out in (64 * MB, 64 * MB + cache - item, 64 * MB - out_bytes + item):
        caches = {"k": 64 * MB, "v": 128 * MB} if which == "k" else {"k": 128 * MB, "v": 64 * MB}
        assert "apart from the cache" in refusal("ferris_tree_attention", attention(dtype, MB, out, **caches))


PLACES = dict(probs=MB, draft=2 * MB, tokens=3 * MB, parents=4 * MB, q_start=5 * MB, uniforms=6 * MB, nodes=7 * MB, accepted=8 * MB, token=9 * MB, ldp=110, ldd=120,
              seqs=2, rows=3, vocab=100, width=4)


@pytest.mark.parametrize("changes", [dict(accepted=9 * MB), dict(accepted=9 * MB + 4), dict(token=7 * MB + 28), dict(nodes=8 * MB - 28), dict(nodes=9 * MB + 4)])
def test_a_verification_that_writes_twice_in_one_place_is_refused(changes):
    assert "apart from one another" in refusal("ferris_verify_tree", verification_arguments(**{**PLACES, **changes}))


@pytest.mark.parametrize("read, end", [("probs", 4 * 320), ("draft", 4 * 340), ("tokens", 12), ("parents", 12), ("uniforms", 12), ("q_start", 12)])
@pytest.mark.parametrize("output, size", [("nodes", 32), ("accepted", 8), ("token", 8)])
def test_a_verification_into_what_it_reads_is_refused(read, end, output, size):
    for at in (PLACES[read], PLACES[read] + end - 4, PLACES[read] - size + 4):
        assert "apart from what is read" in refusal("ferris_verify_tree", verification_arguments(**{**PLACES, output: at}))
