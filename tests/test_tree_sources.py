"""The operators over trees of drafted tokens as far as they show without a GPU: what they refuse, how work is dealt out, what their kernels keep to."""

import random
import re

import pytest
import torch

from test_kernel_sources import CSRC, kernels_with

PAGE = 1 << 20  # an address that nothing is read from: every call here is refused, or has nothing to do
BF16, FP32 = torch.bfloat16, torch.float32


def library():
    from ferrisinfer_b200.kernels import ops

    return ops, ops._lib()


def refusal(entry, arguments):
    """What the library says when it refuses."""
    ops, lib = library()
    assert getattr(lib, entry)(arguments) != 0
    return lib.ferris_last_error().decode()


# ------------------------------------------------------------------------------------------------ refusals
def attention_arguments(**changes):
    ops, _ = library()
    a = dict(q=PAGE, out=PAGE, k=PAGE, v=PAGE, tables=PAGE, q_start=PAGE, start_row=PAGE, parents=PAGE, parts=PAGE, stream=0, ldq=256, ldo=256,
             dtype=ops._DT[BF16], pages=4, kv_heads=2, page_size=16, head_dim=64, width=4, seqs=1, tokens=3, heads=4, max_nodes=3, max_kv=40, window=0, scale=0.125)
    a.update(changes)
    return ops._TREE_ATTENTION.pack(*a.values())


@pytest.mark.parametrize("changes, said", [
    (dict(heads=3), "3 heads over 2 kv heads"), (dict(kv_heads=0), "kv heads"), (dict(head_dim=12), "multiple of 8"), (dict(head_dim=264), "at most 256"),
    (dict(head_dim=0), "multiple of 8"), (dict(max_nodes=257), "at most 256 tokens"), (dict(pages=0), "0 pages"), (dict(page_size=0), "pages of 0 rows"),
    (dict(width=0), "tables of 0 blocks"), (dict(max_kv=0), "0 rows at most"), (dict(k=PAGE + 8), "16 bytes"), (dict(v=PAGE + 2), "16 bytes"),
    (dict(parts=0), "scratch"), (dict(parts=PAGE + 4), "scratch"), (dict(seqs=1 << 30, kv_heads=64, heads=64, max_kv=1 << 24, width=1 << 20), "exceed one launch"),
    (dict(max_kv=0x7fffffff, width=2, page_size=1 << 30), "rows, not"),
])
@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
def test_attention_is_refused(dtype, changes, said):
    ops, _ = library()
    assert said in refusal("ferris_tree_attention", attention_arguments(dtype=ops._DT[dtype], **changes))


@pytest.mark.parametrize("changes", [dict(seqs=0), dict(tokens=0), dict(max_nodes=0)])
def test_attention_of_nothing_does_nothing(changes):
    _, lib = library()
    assert lib.ferris_tree_attention(attention_arguments(**changes)) == 0


def rows_arguments(**changes):
    ops, _ = library()
    a = dict(layers=PAGE, tables=PAGE, start_row=PAGE, nodes=PAGE, accepted=PAGE, stream=0, num_layers=2, pages=4, kv_heads=2, page_size=16, row_bytes=128, align=16,
             width=4, seqs=1, path=5)
    a.update(changes)
    return ops._TREE_ROWS.pack(*a.values())


@pytest.mark.parametrize("changes, said", [
    (dict(path=257), "at most 256 nodes"), (dict(pages=0), "0 pages"), (dict(kv_heads=0), "0 heads"), (dict(page_size=0), "of 0 rows"), (dict(row_bytes=0), "0 bytes"),
    (dict(width=0), "0 blocks"), (dict(seqs=65536), "65536 requests"), (dict(row_bytes=129), "rows of 129 bytes"), (dict(align=1), "multiple of 1"),
])
def test_moves_are_refused(changes, said):
    assert said in refusal("ferris_tree_rows", rows_arguments(**changes))


@pytest.mark.parametrize("changes", [dict(seqs=0), dict(num_layers=0), dict(path=1), dict(path=0)])
def test_moves_of_nothing_do_nothing(changes):
    _, lib = library()
    assert lib.ferris_tree_rows(rows_arguments(**changes)) == 0


def verification_arguments(**changes):
    ops, _ = library()
    a = dict(probs=PAGE, draft=0, tokens=PAGE, parents=PAGE, q_start=PAGE, uniforms=PAGE, nodes=PAGE, accepted=PAGE, token=PAGE, stream=0, ldp=100, ldd=0, seqs=1,
             rows=3, vocab=100, width=4)
    a.update(changes)
    return ops._VERIFY_TREE.pack(*a.values())


@pytest.mark.parametrize("changes", [dict(vocab=0), dict(rows=-1), dict(width=0), dict(ldp=99), dict(draft=PAGE, ldd=99)])
def test_verification_is_refused(changes):
    assert "probabilities" in refusal("ferris_verify_tree", verification_arguments(**changes))


def test_verification_of_nothing_does_nothing():
    _, lib = library()
    assert lib.ferris_verify_tree(verification_arguments(seqs=0)) == 0


@pytest.mark.parametrize("vocab, ldl, ldo, said", [(0, 8, 8, "vocabulary 0"), (9, 8, 9, "row strides 8 and 9"), (9, 9, 8, "row strides 9 and 8"),
                                                   (524289, 524289, 524289, "at most 524288")])
def test_probabilities_are_refused(vocab, ldl, ldo, said):
    _, lib = library()
    assert lib.ferris_sampling_probs(PAGE, ldl, PAGE, ldo, 1, vocab, None, None, None, None) != 0
    assert said in lib.ferris_last_error().decode()
    assert lib.ferris_sampling_probs(PAGE, ldl, PAGE, ldo, 0, vocab, None, None, None, None) == 0


def test_tensors_of_the_host_are_refused():
    ops, _ = library()
    x, i, f = torch.zeros(2, 128), torch.zeros(2, dtype=torch.int32), torch.zeros(2)
    cache = torch.zeros(1, 1, 16, 64)
    table = torch.zeros(2, 1, dtype=torch.int32)
    calls = [lambda: ops.tree_attention(x, x.clone(), cache, cache, table, torch.zeros(3, dtype=torch.int32), i, i, 1, 16, 2, 0.1),
             lambda: ops.sampling_probs(x, x.clone()), lambda: ops.verify_tree(x, i, i, i, f, table, i, i),
             lambda: ops.CacheLayers([(cache, cache)])]
    for call in calls:
        with pytest.raises(ops.KernelError, match="CUDA|GPU"):
            call()


# ------------------------------------------------------------------------------------------------ how work is dealt out
SMS = 148  # what the library takes where it finds no GPU


def variant(dtype, D, rows, page_size):
    """(cached rows of a tile, query rows of a block, blocks on an SM, flat) of the kernels, where they are of one size."""
    if dtype == FP32 and D > 128:
        return 32, 64, 1, True
    if dtype == FP32:
        return 64, 32 if -(-rows // 32) * 32 < -(-rows // 64) * 64 else 64, 1, True
    assert rows > 16 and page_size % 16 == 0 and D in (64, 128)  # (on tcgen05, where the step is long or the rows are many)
    return 128, 256 if rows > 128 else 128, 1 if rows > 128 else 2, False


def deal(seqs, kv_heads, group, max_nodes, max_kv, unit, rows, blocks, flat):
    row_blocks = -(-max_nodes * group // rows)
    lanes = 1 if flat else row_blocks
    most = seqs * kv_heads * (row_blocks if flat else 1) * (-(-max_kv // unit) + 1)
    return max(1, min(SMS * blocks // lanes, most)), lanes


@pytest.mark.parametrize("dtype, D, page_size", [(BF16, 64, 16), (BF16, 128, 64), (FP32, 64, 16), (FP32, 96, 5), (FP32, 256, 16)])
@pytest.mark.parametrize("seqs, kv_heads, group, max_nodes, max_kv", [(1, 2, 7, 16, 1000), (64, 4, 7, 64, 4161), (1, 1, 16, 256, 100000), (300, 8, 1, 40, 33), (6, 2, 6, 13, 1546)])
def test_scratch_has_room_for_the_parts_and_no_more(dtype, D, page_size, seqs, kv_heads, group, max_nodes, max_kv):
    ops, lib = library()
    unit, rows, blocks, flat = variant(dtype, D, max_nodes * group, page_size)
    groups, lanes = deal(seqs, kv_heads, group, max_nodes, max_kv, unit, rows, blocks, flat)
    floats = ops._tree_attention_scratch(ops._DT[dtype], D, seqs, kv_heads, group, max_nodes, max_kv, page_size, 10 ** 6, 0.1, 0, 0)
    assert floats == 2 * groups * lanes * rows * (D + 2) + 4 * groups


@pytest.mark.parametrize("seed", range(300))
def test_every_part_has_a_place_of_its_own_and_is_joined(seed):
    """The dealing out of tiles, step by step: every tile once, no two parts in one place, and the join reads those that were left and no others."""
    rng = random.Random(seed)
    kv_heads, group, flat = rng.choice([1, 2, 4, 8]), rng.choice([1, 4, 7]), rng.random() < 0.5
    unit, rows = rng.choice([(64, 32), (64, 64), (128, 128), (128, 256), (32, 16)])
    seqs, most = rng.choice([1, 2, 7, 40, 200]), rng.choice([1, 60, 1000, 30000])
    requests = [(rng.choice([0, 1, 1, 5, 33, 64]), rng.randint(0, most)) for _ in range(seqs)]
    max_nodes, max_kv = max(max(n for n, _ in requests), 1), max(max(s + n for n, s in requests), 1)
    groups, lanes = deal(seqs, kv_heads, group, max_nodes, max_kv, unit, rows, 1, flat)
    items = []  # [request, kv head, block, tiles, first place]
    for r, (n, start) in enumerate(requests):
        for h in range(kv_heads if n else 0):
            for b in range(-(-n * group // rows) if flat else 1):
                items.append([r, h, b, max(-(-(start + n) // unit), 1)])
    total = sum(i[3] for i in items)
    per, more = divmod(total, groups)
    runs, even = 1, -(-total // groups)  # tiles of a run of one item; 1: none
    for u in range(even, even + 2 if even > 1 else 0):
        if seqs <= 128 and sum(-(-i[3] // u) for i in items) <= groups:
            runs, per, more = u, u, 0
            break
    places_used = 0
    for i in items:
        i.append(places_used)
        places_used += -(-i[3] // runs) * runs
    begins = lambda g: min(places_used, g * per + min(g, more))
    owner = lambda t: t // (per + 1) if t < more * (per + 1) else more + (t - more * (per + 1)) // per
    places, begun, done = {}, {}, 0
    for g in range(groups):
        lo, hi, segments = begins(g), begins(g + 1), 0
        for item in items:
            first, last = max(lo - item[4], 0), min(hi - item[4], item[3])
            if first >= last:
                continue
            done, segments = done + last - first, segments + 1
            assert all(owner(item[4] + t) == g for t in (first, last - 1))
            if first or last < item[3]:
                assert (g, first == 0) not in places
                places[g, first == 0] = item
            if first == 0 and last < item[3]:
                assert g not in begun
                begun[g] = (item, owner(item[4] + item[3] - 1))
        assert hi - lo <= even + 1 and (runs == 1 or segments <= 1)
    assert done == total
    joined = {}
    for g, (item, end) in begun.items():
        for k in range(end - g + 1):
            joined[g + k, k == 0] = item
    assert joined == places


# ------------------------------------------------------------------------------------------------ what the kernels keep to
def test_tensor_memory_is_allocated_before_dependents_are_let_in():
    found = kernels_with("tensor_memory_take")
    assert {k for _, k, _ in found} == {"tree_attention_tc_kernel"}
    for file, kernel, body in found:
        allocated = body.index("tensor_memory_take")
        assert "pdl_launch_dependents()" not in body[:allocated]
        assert body.count("return;") == body.count("if (node < 0) return;"), f"{file}: {kernel} could leave with its tensor memory"  # (in a lambda)
        assert "tmem_dealloc" in body[allocated:]


def test_waits_have_limits():
    for _, kernel, body in kernels_with("tensor_memory_take"):
        assert "try_wait" not in body and "mbar_wait(" in body
        assert not re.search(r"\bbreak;", body), f"{kernel}: a loop that ends early could leave others at a barrier of some of the warps"


def test_registers_that_warps_take_are_those_the_block_was_launched_with():
    source = open(f"{CSRC}/tree_attention_tc.cu").read()
    given = {k: int(v) for k, v in re.findall(r"(LAUNCH_REGISTERS|SOFTMAX_REGISTERS|OTHER_REGISTERS) = (\d+)", source)}
    assert 2 * given["SOFTMAX_REGISTERS"] + given["OTHER_REGISTERS"] <= 3 * given["LAUNCH_REGISTERS"]
    assert 3 * 128 * given["LAUNCH_REGISTERS"] <= 65536 and all(v % 8 == 0 for v in given.values())
    assert "registers < LAUNCH_REGISTERS" in source  # (asked of the kernel that was built, before it is launched)


@pytest.mark.parametrize("file", ["tree_attention_f32.cu", "tree_attention_mma.cu", "sampling_probs.cu"])
def test_shared_memory_that_is_read_by_16_bytes_begins_on_16(file):
    found = re.findall(r"extern __shared__ ([^;]*);", open(f"{CSRC}/{file}").read())
    assert found and all("__align__(16)" in one or "__align__(128)" in one for one in found), found
