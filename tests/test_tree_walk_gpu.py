"""How the work of a step of trees is dealt out, as the kernels' own ``TreeWalk`` does it (compiled into ``tree_walk.cu``): every tile that a node can see goes to one
group of blocks, no two parts have one place, and the groups' notes lead the join to the parts that were left and to no others."""

import ctypes
import os
import random
import subprocess

import pytest
import torch

from test_tree_gpu import DEV, ints

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tree_walk(tmp_path_factory):
    from ferrisinfer_b200.kernels import build

    here, out = os.path.dirname(os.path.abspath(__file__)), str(tmp_path_factory.mktemp("walk") / "tree_walk.so")
    subprocess.run([build._find_nvcc(), *build.ARCH_FLAGS, *build.NVCC_FLAGS, "-I", build.CSRC, "-shared", os.path.join(here, "tree_walk.cu"), "-o", out], check=True)
    entry = ctypes.CDLL(out).tree_walk
    entry.argtypes = [ctypes.c_int] * 7 + [ctypes.c_void_p] * 3 + [ctypes.c_int] * 7
    return entry


def case(seed):
    draw = random.Random(seed)
    c = {"kv_heads": draw.choice([1, 2, 4, 8]), "group": draw.choice([1, 4, 7]), "flat": draw.random() < 0.5}
    c["unit"], c["rows"] = draw.choice([(64, 32), (128, 16), (128, 128), (128, 256)])
    seqs, most = draw.choice([1, 2, 7, 40, 127, 128, 129, 200]), draw.choice([1, 60, 1000, 30000])
    c["requests"] = [(draw.choice([0, 1, 1, 5, 33, 64]), draw.randint(0, most)) for _ in range(seqs)]
    if draw.random() < 0.2:
        c["requests"][draw.randrange(seqs)] = (5, 0x7fffffff)  # says that it has more rows than there are
    c["max_nodes"] = max(max(n for n, _ in c["requests"]), 1)
    longest = max(s + n for n, s in c["requests"] if s < 1 << 30) if any(s < 1 << 30 for _, s in c["requests"]) else 1
    c["limit"] = max(1, draw.choice([longest, longest, longest // 2, longest + 1000]))
    c["window"] = draw.choice([0, 0, 1, 40, 128, 1000, 0x7fffffff])
    items = lambda: sum(-(-n * c["group"] // c["rows"]) for n, _ in c["requests"]) * c["kv_heads"]
    while items() > 2000:
        c["requests"] = c["requests"][::2]
    c["items"] = items()
    row_blocks = -(-c["max_nodes"] * c["group"] // c["rows"])
    c["lanes"] = 1 if c["flat"] else row_blocks
    c["groups"] = draw.choice([1, 2, 13, 148, 296, max(1, 148 // c["lanes"])])
    return c


def walked(tree_walk, c):
    """(segments, note) of every block."""
    q_start = [0]
    for n, _ in c["requests"]:
        q_start.append(q_start[-1] + n)
    starts, q_start_there = ints([s for _, s in c["requests"]]), ints(q_start)
    blocks, room = (c["groups"] + 3) * c["lanes"], c["items"] + 1  # (three groups more than there are)
    out = torch.full((blocks, 5 + 8 * room), -7, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    assert tree_walk(c["unit"], c["rows"], c["flat"], blocks, c["groups"], c["lanes"], room, out.data_ptr(), q_start_there.data_ptr(), starts.data_ptr(), len(c["requests"]),
                     q_start[-1], c["kv_heads"], c["group"], c["max_nodes"], c["limit"], c["window"]) == 0
    result = []
    most = int(out[:, 0].max())
    assert most < room
    for row in out[:, :5 + 8 * most].tolist():
        result.append(([tuple(row[5 + 8 * i:13 + 8 * i]) for i in range(row[0])], row[1:5]))
    return result


@pytest.mark.parametrize("seed", range(120))
def test_every_tile_goes_to_one_group_and_every_part_is_joined(tree_walk, seed):
    c = case(seed)
    unit, rows, lanes, groups = c["unit"], c["rows"], c["lanes"], c["groups"]
    blocks = walked(tree_walk, c)
    places, notes, seen = {}, {}, {}
    for b, (segments, note) in enumerate(blocks):
        g, lane = divmod(b, lanes)
        if g >= groups:
            assert not segments and note[0] == -1  # (they would have no place)
        noted = None
        for seq, head, block, first, last, tiles, low, start in segments:
            assert 0 <= first < last <= tiles and (c["flat"] or block == lane)
            item = (seq, head, block)
            seen.setdefault(item, []).append((first, last, tiles, low, g))
            if first or last < tiles:
                assert (b, first == 0) not in places, "two parts in one place"
                places[b, first == 0] = item
            if first == 0 and last < tiles:
                assert noted is None
                noted = item
        assert (note[0] >= 0) == (noted is not None)
        if noted:
            assert tuple(note[:3]) == noted
            if lane == 0:
                notes[g] = note
    # every item that there is, whole, in the order of the groups, and all that one of its nodes can see
    expected = set()
    for seq, (n, start) in enumerate(c["requests"]):
        for block in range(-(-n * c["group"] // rows)):
            expected |= {(seq, head, block) for head in range(c["kv_heads"])}
    assert set(seen) == expected
    for (seq, _, _), parts in seen.items():
        n, start = c["requests"][seq]
        there = min(start + n, c["limit"])
        at = 0
        for first, last, tiles, low, g in sorted(parts, key=lambda p: p[4]):
            assert first == at
            at = last
        assert at == tiles and len({p[2:4] for p in parts}) == 1 and len({p[4] for p in parts}) == len(parts)
        assert (low + tiles) * unit >= there
        assert low * unit <= (max(0, start - c["window"] + 1) if c["window"] else 0)
    # the join: from a note on, the groups up to the one that it names; a lane's block of query rows where there are lanes
    joined = {}
    for g, (seq, head, block, end) in notes.items():
        for lane in range(lanes):
            item = (seq, head, lane if lanes > 1 else block)
            if item not in seen:
                continue  # (a request with fewer query rows)
            for k in range(end - g + 1):
                joined[(g + k) * lanes + lane, k == 0] = item
    assert joined == places
