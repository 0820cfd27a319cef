"""What the packed cache's kernels lay out, as far as it shows without a GPU."""

import ctypes
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ferrisinfer_b200", "csrc")


@pytest.mark.parametrize("file", ["packed_cache.cu", "packed_attention.cu"])
def test_shared_memory_that_is_read_by_16_bytes_begins_on_16(file):
    """Dynamic shared memory stands behind the static: where it begins is the declaration's alignment, and no more."""
    source = open(os.path.join(CSRC, file)).read()
    found = re.findall(r"extern __shared__ ([^;]*);", source)
    assert found and all("__align__(16)" in one for one in found), found


def _library():
    from ferrisinfer_b200.kernels import build

    return build.load_library()


SMS = 148  # what the library takes where it finds no GPU


def part_places(pairs, kv_heads, max_kv):
    """(grid, places for parts) of a step of prompts."""
    grid = min(SMS + pairs * kv_heads, pairs * kv_heads * (max_kv // 128 + 2))
    return grid, max(grid, 2 * min(grid, SMS))


@pytest.mark.parametrize("seqs, q_len, heads, kv_heads, start", [(4, 2048, 28, 4, 0), (1, 8192, 64, 8, 0), (1, 512, 28, 4, 32768), (6, 700, 12, 2, 0)])
def test_scratch_of_prompts_has_room_for_the_parts_and_no_more(seqs, q_len, heads, kv_heads, start):
    group, D = heads // kv_heads, 128
    needs = (ctypes.c_longlong * 3)()
    plan = _library().ferris_packed_attention_plan
    plan(_bf16(), D, seqs, kv_heads, group, seqs * q_len, q_len, start + q_len, 0, needs)
    pairs = min(seqs * q_len * group // 256 + seqs, seqs * -(-q_len * group // 256))
    grid, places = part_places(pairs, kv_heads, start + q_len)
    operands, parts = pairs * kv_heads * 2 * (2 * 16384 + 4096), places * (D + 2) * 256 * 4
    few = 2 * (SMS * 2 + seqs * kv_heads) * 8 * (D + 2) * 4  # parts of requests with few rows beside them
    rest = needs[0] * 4 - operands - parts
    assert 0 <= rest <= pairs * kv_heads * 4096 + few + 16 * 1024, (needs[0] * 4, operands, parts, rest)


def _bf16():
    from ferrisinfer_b200.kernels import ops

    import torch

    return ops._DT[torch.bfloat16]


@pytest.mark.parametrize("seed", range(300))
def test_every_part_of_a_prompt_has_a_place_of_its_own(seed):
    """The dealing out of blocks of cached rows, step by step: no two parts in one place, none outside the scratch."""
    import random

    rng = random.Random(seed)
    kv_heads, most = rng.choice([1, 2, 4, 8]), rng.choice([3, 40, 400, 4000])
    counts = [rng.randint(1, most) for _ in range(rng.choice([1, 2, 7, 60, 300]))]
    if rng.random() < 0.3:
        counts = [most] * len(counts)
    grid, room = part_places(len(counts), kv_heads, max(counts) * 128)
    units = sum(counts) * kv_heads
    chunk = max(4, -(-units // SMS))
    while chunk < 16 and len(counts) * kv_heads <= SMS and sum(-(-c // chunk) for c in counts) * kv_heads > SMS:
        chunk += 1
    blocks, runs = min(SMS, max(1, units // 4)), chunk >= 16
    block_of = lambda u: ((u + 1) * blocks - 1) // units
    taken, u, block = set(), 0, 0
    for c in counts:
        for _ in range(kv_heads):
            if runs:
                first, last = block_of(u), block_of(u + c - 1)
                places = [2 * i + (i == first) for i in range(first, last + 1)]
                u += c
            else:
                n = -(-c // chunk)
                first, last = block, block + n - 1
                places = list(range(first, last + 1))
                block += n
            assert last < grid
            if first != last:
                assert not taken & set(places) and max(places) < room
                taken |= set(places)
