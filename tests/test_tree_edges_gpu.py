"""Operators of steps over drafted tokens at the edges of what they take."""

import math

import pytest
import torch

import plain_tree as plain
from test_tree_gpu import DEV, Step, ints, nothing_reported, ops, rng, run_verify, workspace  # noqa: F401  (fixtures among them)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ probabilities
def in_64_bits(logits, temperature, top_k, top_p, rows=32):
    """(first row, probabilities) of some rows at a time; logits without NaN."""
    place = torch.arange(logits.shape[1], device=DEV)
    for first in range(0, len(logits), rows):
        x = logits[first:first + rows].double()
        T, k, p = (torch.tensor(o[first:first + rows], dtype=torch.float32, device=DEV).double()[:, None] for o in (temperature, top_k, top_p))
        x, order = torch.sort(x, dim=1, descending=True, stable=True)
        w = torch.where((k <= 0) | (place < k), torch.exp((x - x[:, :1]) / T), 0.0)
        w = torch.where((p >= 1) | (place == 0) | (torch.cumsum(w, 1) - w < p * w.sum(1, keepdim=True)), w, 0.0)
        yield first, torch.zeros_like(x).scatter_(1, order, w / w.sum(1, keepdim=True))


@pytest.mark.parametrize("V", [262143, 262144, 524287, 524288])
@pytest.mark.parametrize("top_k, top_p", [(0, 0.5), (0, 0.999), (0, 1e-6), (1000, 0.5), (400000, 0.75), (20, 0.5), (0, 1.0)])
def test_equal_logits_of_the_largest_vocabularies(ops, V, top_k, top_p):
    """The row's mass is as many times the greatest weight as it has tokens.  A row of one logit, of minus infinity, of NaN, and one whose temperature makes all weights equal."""
    logits = torch.full((4, V), 1.5, device=DEV)
    logits[1], logits[2] = -math.inf, math.nan
    logits[3] = torch.randn(V, generator=rng(1), device=DEV)
    out = torch.full((4, V), 9.0, device=DEV)
    p = torch.tensor(top_p, dtype=torch.float32)
    ops.sampling_probs(logits, out, torch.tensor([1.0, 1.0, 1.0, 1e30], device=DEV), ints([top_k] * 4), p.to(DEV).repeat(4))
    count = min(top_k, V) if top_k else V
    count = math.ceil(p.double().item() * count) if top_p < 1 else count  # (the product of 24 and 19 bits is exact)
    want = torch.zeros(4, V, dtype=torch.float64, device=DEV)
    want[:3, :count] = 1 / count
    want[3, torch.sort(logits[3], descending=True, stable=True).indices[:count]] = 1 / count
    assert torch.equal(out > 0, want > 0)
    assert ((out - want).abs() <= 2.0 ** -22 / count).all()  # the sum of equal numbers, a quotient and its rounding, a product


@pytest.mark.parametrize("V", [151936, 524288])
@pytest.mark.parametrize("depth", [30.0, 32.0, 40.0])
def test_masses_that_are_nothing_one_by_one(ops, V, depth):
    """Two great logits and a long flat tail below them: a weight is a whole number of 2^-45 of the greatest (2^-44 from 2^19 tokens on), so that n tokens' mass
    is off by n times half of that at most, and each weight by 2^-46 of itself.  Who stays is right for some mass within that bound."""
    logits = torch.full((2, V), -depth, device=DEV)
    logits[:, V // 3], logits[:, V // 2] = 0.0, 0.0
    logits[1, ::2] -= 0.25
    logits[1, V // 3] = logits[1, V // 2] = 0.0
    for top_p in (0.5, 0.49999997, 0.50000006, 0.99999994):
        out = torch.full((2, V), 9.0, device=DEV)
        p = torch.tensor([top_p] * 2, dtype=torch.float32, device=DEV)
        ops.sampling_probs(logits, out, torch.ones(2, device=DEV), None, p)
        order = torch.sort(logits, dim=1, descending=True, stable=True).indices
        w = torch.exp(logits.double()).gather(1, order)
        kept = out.gather(1, order) > 0
        count = kept.sum(1, keepdim=True)
        assert torch.equal(kept, torch.arange(V, device=DEV) < count)  # the first ones
        upto = torch.cumsum(w, 1)
        aim, bound = p.double()[:, None] * upto[:, -1:], V * 2.0 ** (-46 if V < 1 << 19 else -45) + upto[:, -1:] * 2.0 ** -45
        assert (upto.gather(1, count - 1) >= aim - bound).all()
        assert ((count == 1) | (upto.gather(1, (count - 2).clamp(min=0)) < aim + bound)).all()


BATCHES = {
    "plain": [(1.0, 0, 1.0)], "chat": [(0.7, 20, 0.9)], "mass": [(0.8, 0, 0.9)],
    "mixed": [(1.0, 0, 1.0), (0.7, 20, 0.9), (0.8, 0, 0.9), (1.0, 3001, 0.95), (0.6, 50, 1.0), (1.3, 0, 0.5)],
}


@pytest.mark.parametrize("options", BATCHES.values(), ids=BATCHES.keys())
def test_probabilities_of_a_busy_server(ops, options):
    """512 rows of 151,936, a few likely tokens in each, against 64 bits on the same logits."""
    n, V = 512, 151936
    gen = rng(41)
    logits = torch.randn(n, V, generator=gen, device=DEV) * 2
    likely = torch.arange(20, device=DEV) * (V // 20) + torch.randint(V // 20, (n, 20), generator=gen, device=DEV)  # (no place twice)
    logits.scatter_(1, likely, 6 + 2 * torch.randn(n, 20, generator=gen, device=DEV))
    temperature, top_k, top_p = ([options[i % len(options)][j] for i in range(n)] for j in range(3))
    out = torch.full((n, V), 9.0, device=DEV)
    ops.sampling_probs(logits, out, torch.tensor(temperature, device=DEV), ints(top_k), torch.tensor(top_p, device=DEV))
    for first, ref in in_64_bits(logits, temperature, top_k, top_p):
        got, x = out[first:first + len(ref)].double(), logits[first:first + len(ref)].double()
        assert torch.equal(got > 0, ref > 0)
        # an exponent of 32 bits is off by 2^-23 of itself, the exponential, the sum and the quotient by a few 2^-24
        exponent = (x.amax(1, keepdim=True) - x) / torch.tensor(temperature[first:first + len(ref)], device=DEV).double()[:, None]
        assert ((got - ref).abs() <= ref * (exponent * 2.0 ** -22 + 2.0 ** -19) + 1e-37).all()


# ------------------------------------------------------------------------------------------------ verification
TOP = 1 - 2.0 ** -24  # the greatest random number


@pytest.mark.parametrize("rows, tokens, parents, u, path, token", [
    # two tokens are all that the row has, of which the last random number refuses both: 1 - 0.6 is a little more than the second's
    ([[0.6, 0.39999995, 0.0]], [0, 0, 1], [-1, 0, 0], [0.5, TOP, TOP], [0], 1),
    # (the other way round the second one is accepted: (1 - 2^-24) (1 - 0.39999994636) = 0.60000001788 < 0.60000002384, and its row has nothing)
    ([[0.6, 0.39999995, 0.0]], [0, 1, 0], [-1, 0, 0], [0.5, TOP, TOP], [0, 2], -1),
    # a row whose probabilities do not add up to one
    ([[0.0, 0.25, 0.0]], [0, 1, 2], [-1, 0, 0], [0.0, 0.5, 0.5], [0], 1),
    ([[0.0, 0.25, 0.0]], [0, 1, 1], [-1, 0, 0], [0.0, 0.5, 0.0], [0], 1),
    # on the second node of a path
    ([[0.0, 1.0, 0.0], [0.0, 0.0, 0.75]], [0, 1, 2], [-1, 0, 1], [0.3, 0.5, 0.875], [0, 1], 2),
    # what was refused before the path went on is forgotten
    ([[0.5, 0.5, 0.0], [0.0] * 3, [0.0] * 3], [0, 0, 1], [-1, 0, 0], [0.3, 0.875, 0.25], [0, 2], -1),
    # nothing that could be refused
    ([[0.0, 0.0, 0.0]], [0, 1, 2], [-1, 0, 0], [0.3, 0.5, 0.5], [0], -1),
])
def test_chosen_drafts_that_are_all_refused(ops, rows, tokens, parents, u, path, token):
    """Where refusals have left nothing of a row, the token refused last of those that had a probability follows, as it would if the row added up to one."""
    n = len(tokens)
    for V in (3, 700):
        probs = torch.zeros(n, V, device=DEV)
        for i, row in enumerate(rows):
            probs[i, :3] = torch.tensor(row, device=DEV)
        got = run_verify(ops, probs, tokens, parents, [0, n], u, 3)
        assert got == ([path + [-1] * (3 - len(path))], [len(path) - 1], [token])


# ------------------------------------------------------------------------------------------------ memory that is shared
def test_attention_into_memory_that_it_reads_is_refused(ops, workspace):
    from ferrisinfer_b200.errors import KernelError

    step = Step(torch.bfloat16, 4, 2, 64, 16, [3, 2], [20, 30], extra_columns=512)
    want = step.run(ops, workspace).clone()
    call = lambda q, out: ops.tree_attention(q, out, step.k, step.v, *step.device_tensors, *step.most, 4, 0.125, workspace=workspace)
    flat = torch.zeros(6 * 768, dtype=torch.bfloat16, device=DEV)
    rows = flat[:5 * 768].view(5, 768)
    rows.copy_(step.q)
    for q, out in ((rows, rows[:, :256]), (rows, rows[:, 255:511]), (rows[:, 200:456], rows[:, :256]),
                   (rows, flat[64:64 + 5 * 256].view(5, 256)),                   # rows of another length
                   (rows, flat.as_strided((5, 256), (768, 1), 700)),             # from the end of a row to the beginning of the next one
                   (step.q, step.k.view(-1)[:5 * 256].view(5, 256)), (step.q, step.v.view(-1)[-5 * 256:].view(5, 256))):
        with pytest.raises(KernelError, match="apart"):
            call(q, out)
    call(rows, rows[:, 256:512])  # columns beside the queries', in the same rows, are apart from them
    assert torch.equal(rows[:, 256:512], want) and torch.equal(rows[:, :256], step.q[:, :256])
    call(rows[:, :256], rows[:, 512:])
    assert torch.equal(rows[:, 512:], want)


def test_verification_into_memory_that_it_reads_or_twice_is_refused(ops):
    from ferrisinfer_b200.errors import KernelError

    i32 = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=DEV)
    probs, one = torch.full((5, 30), 1 / 30, device=DEV), ints([0, 2, 5])
    both = i32(4)
    good = dict(probs=probs, tokens=i32(5), parents=i32(5) - 1, seq_q_start=one, uniforms=torch.zeros(5, device=DEV), out_nodes=i32(2, 2), out_accepted=i32(2), out_token=i32(2))
    ops.verify_tree(**good)
    for change in (dict(out_accepted=both[:2], out_token=both[1:3]), dict(out_nodes=both.view(2, 2), out_token=both[2:]), dict(out_token=good["tokens"][3:]),
                   dict(out_accepted=good["parents"][:2]), dict(out_nodes=probs.view(torch.int32)[0, :4].view(2, 2)), dict(out_token=one[1:]),
                   dict(out_token=good["uniforms"].view(torch.int32)[:2])):
        with pytest.raises(KernelError, match="apart"):
            ops.verify_tree(**{**good, **change})
    ops.verify_tree(**{**good, "out_accepted": both[:2], "out_token": both[2:]})


def test_cache_layers_that_share_memory_are_refused(ops):
    from ferrisinfer_b200.errors import KernelError

    cache = torch.zeros(2, 4, 2, 16, 8, device=DEV)
    flat = torch.zeros(2 * 4 * 2 * 16 * 8, device=DEV)
    k, v = cache
    ops.CacheLayers([(k, v)])
    for layers in ([(k, k)], [(k, v), (v, k.clone())], [(k, v), (k, v)], [(flat[:1024].view(4, 2, 16, 8), flat[8:1032].view(4, 2, 16, 8))]):
        with pytest.raises(KernelError, match="share memory"):
            ops.CacheLayers(layers)
    ops.CacheLayers([(flat[:1024].view(4, 2, 16, 8), flat[1024:].view(4, 2, 16, 8))])


# ------------------------------------------------------------------------------------------------ attention
def test_attention_without_any_cached_row_is_refused(ops, workspace):
    from ferrisinfer_b200.errors import KernelError

    step = Step(torch.bfloat16, 4, 2, 64, 16, [3, 2], [20, 30])
    step.run(ops, workspace)
    tables, *others = step.device_tensors
    out = torch.full((5, 256), 7.0, dtype=torch.bfloat16, device=DEV)
    call = lambda k, tables, most: ops.tree_attention(step.q, out, k, k, tables, *others, *most, 4, 0.125, workspace=workspace)
    for k, t, most in ((step.k, tables, (3, 0)), (step.k[:0], tables, (3, 40)), (step.k, tables[:, :0].contiguous(), (3, 40))):
        with pytest.raises(KernelError, match="no rows"):
            call(k, t, most)
    call(step.k, tables, (0, 0))  # (no nodes either)
    assert (out == 7).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("nodes", [[5, 12], [5, 70]])
def test_texts_beyond_their_tables(ops, workspace, dtype, window, nodes):
    """A request that says it has more rows than its table sees those that the table has, behind a window none; the other request is none the wiser."""
    step = Step(dtype, 12, 2, 64, 16, nodes, [60, 200])
    for t, seed in ((step.k, 5), (step.v, 6)):  # (what lies on the tables' last rows is seen now)
        t.copy_(torch.where(torch.isnan(t), torch.randn(t.shape, generator=rng(seed), device=DEV).to(dtype), t))
    most = max(nodes), 200 + nodes[1]
    for start in (0x7fffffff, 1 << 30, 100000):
        step.starts[0] = start
        out = step.run(ops, workspace, window=window, most=most)
        ref, mag, size = plain.tree_attention(step.q, step.k, step.v, step.tables, step.q_start, step.starts, step.parents, 12, 0.125, window, max_rows=most[1])
        step.compare(out, ref, plain.attention_tolerance(dtype, ref, mag, size, most[1], 64))
        assert not window or (out[:5] == 0).all()
        assert window or (out[:5] != 0).any(1).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("heads, kv_heads, D, most_nodes", [(14, 2, 64, 5), (8, 2, 128, 20), (14, 2, 64, 40)])
def test_a_recorded_step_of_a_padded_batch(ops, dtype, heads, kv_heads, D, most_nodes):
    """Recorded once for the most requests, nodes and rows, and replayed with fewer: requests without nodes, query rows that nobody brings.  (5 nodes are 35 query rows
    of a kv head, 20 are 80, 40 are 280.)"""
    from ferrisinfer_b200.engine.workspace import Workspace

    S, ps, most_rows = 6, 16, 640
    T, width, pages = S * most_nodes, most_rows // ps, S * most_rows // ps + 1
    there = {"q": torch.zeros(T, heads * D, dtype=dtype, device=DEV), "out": torch.zeros(T, heads * D, dtype=dtype, device=DEV),
             "k": torch.zeros(pages, kv_heads, ps, D, dtype=dtype, device=DEV), "v": torch.zeros(pages, kv_heads, ps, D, dtype=dtype, device=DEV)}
    indices = [torch.full((S, width), -1, dtype=torch.int32, device=DEV), ints([0] * (S + 1)), ints([0] * S), ints([-1] * T)]
    workspace = Workspace(DEV)
    call = lambda: ops.tree_attention(there["q"], there["out"], there["k"], there["v"], *indices, most_nodes, most_rows, heads, D ** -0.5, workspace=workspace)
    call()
    workspace.pin()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    batches = [([0] * 6, [0] * 6), ([most_nodes] * 6, [600] * 6), ([0, 1, 0, most_nodes, 2, 0], [9, 0, 600, 17, 599, 600]), ([1] * 6, [600, 0, 1, 128, 127, 300]),
               ([0, 0, 0, 0, 0, most_nodes], [600] * 6), ([3, most_nodes, 0, 0, 0, 0], [1, 400, 0, 0, 0, 0])]
    for nodes, starts in batches:
        n = sum(nodes)
        if n:
            step = Step(dtype, heads, kv_heads, D, ps, nodes, starts)
            for t, values in ((there["k"], step.k), (there["v"], step.v)):
                t.fill_(math.nan)
                t[:len(values)] = values
            there["q"].fill_(math.nan)
            there["q"][:n] = step.q
            indices[0].fill_(-1)
            indices[0][:, :len(step.tables[0])] = ints(step.tables)
            indices[2].copy_(ints(starts)), indices[3][:n].copy_(ints(step.parents))
        indices[1].copy_(ints([sum(nodes[:i]) for i in range(S + 1)]))
        there["out"].fill_(7.0)
        graph.replay()
        if n:
            step.check(there["out"][:n])
        assert (there["out"][n:] == 7).all()
