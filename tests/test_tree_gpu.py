"""Steps over drafted tokens against their plain forms in 64 bits: attention of trees, sampling probabilities, verification, rows kept."""

import math
import random

import pytest
import torch

import plain_tree as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from ferrisinfer_b200.kernels import ops as module

    module.require_device()
    return module


@pytest.fixture(autouse=True)
def nothing_reported(ops):
    yield
    torch.cuda.synchronize()
    ops.check_kernel_status()


@pytest.fixture(scope="module")
def workspace():
    from ferrisinfer_b200.engine.workspace import Workspace

    return Workspace(DEV)


def reported(ops, detail):
    """The call before has reported a bad index of this kind; the report is cleared."""
    torch.cuda.synchronize()
    status = ops.kernel_status()
    assert status == (2 << 16) | detail, hex(status)


def rng(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def tree(n, kind, seed=0):
    """Parents of n nodes."""
    draw = random.Random(seed + n)
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "star":
        return [min(i, 1) - 1 for i in range(n)]
    if kind == "roots":  # nodes with nothing but the text above them among others
        return [-1 if i % 3 == 0 else draw.randrange(i) for i in range(n)]
    return [draw.randrange(i) if i else -1 for i in range(n)]


class Step:
    """A step's inputs; pages in no order, what no request's row lies on is NaN."""

    def __init__(self, dtype, heads, kv_heads, D, page_size, nodes, starts, kind="tree", seed=1, extra_columns=0, spare_rows=0, holes=()):
        gen = rng(seed)
        self.heads, self.D, self.page_size = heads, D, page_size
        self.nodes, self.starts = nodes, starts
        lengths = [n + s for n, s in zip(nodes, starts)]
        blocks = [-(-x // page_size) for x in lengths]
        pages = sum(blocks) + 1
        order = torch.randperm(pages, generator=gen, device=DEV).tolist()
        self.tables, at = [], 0
        width = max(max(blocks), 1)
        self.k, self.v = (torch.full((pages, kv_heads, page_size, D), math.nan, dtype=dtype, device=DEV) for _ in range(2))
        for n, b in zip(lengths, blocks):
            table = order[at:at + b]
            at += b
            for r in range(n):
                self.k[table[r // page_size], :, r % page_size] = (torch.randn(kv_heads, D, generator=gen, device=DEV) * 1.2).to(dtype)
                self.v[table[r // page_size], :, r % page_size] = torch.randn(kv_heads, D, generator=gen, device=DEV).to(dtype)
            self.tables.append(table + [-1] * (width - b))
        for s, block in holes:
            self.tables[s][block] = -1
        self.q_start = [0]
        for n in nodes:
            self.q_start.append(self.q_start[-1] + n)
        self.parents = [p for i, n in enumerate(nodes) for p in tree(n, kind, seed + i)] + [-1] * spare_rows
        T = self.q_start[-1] + spare_rows
        self.q = torch.randn(T, heads * D + extra_columns, generator=gen, device=DEV).to(dtype)
        self.most = max(max(nodes), 1), max(max(lengths), 1)

    def run(self, ops, workspace, window=0, out=None, most=None):
        out = torch.full((self.q.shape[0], self.heads * self.D), 7.0, dtype=self.q.dtype, device=DEV) if out is None else out
        most = most or self.most
        for buffer in workspace._buffers.values():  # (what a call finds in its scratch has no effect)
            buffer.fill_(math.nan if buffer.is_floating_point() else 0)
        self.device_tensors = [ints(self.tables), ints(self.q_start), ints(self.starts), ints(self.parents)]
        ops.tree_attention(self.q, out, self.k, self.v, *self.device_tensors, most[0], most[1], self.heads, self.D ** -0.5, window=window, workspace=workspace)
        return out

    def expected(self, window=0, **kw):
        """Outputs in 64 bits, and how far those of the kernels may be off."""
        ref, mag, size = plain.tree_attention(self.q, self.k, self.v, self.tables, self.q_start, self.starts, self.parents, self.heads, self.D ** -0.5,
                                              window, **kw)
        rows = max(n + s for n, s in zip(self.nodes, self.starts))
        return ref, plain.attention_tolerance(self.q.dtype, ref, mag, size, rows, self.D)

    def check(self, out, window=0, **kw):
        self.compare(out, *self.expected(window, **kw))

    def compare(self, out, ref, tol, rows=slice(None)):
        there = ~torch.isnan(ref[rows])
        off = ((out.double().cpu()[rows] - ref[rows]).abs() / tol[rows])[there]
        assert not torch.isnan(off).any() and (off.numel() == 0 or off.max() <= 1), f"off by {off.max():.3f} of the tolerance"


GEOMETRIES = [  # heads, kv heads, D, page size
    (14, 2, 64, 16), (12, 2, 128, 16), (28, 4, 128, 64), (16, 16, 64, 32), (24, 2, 64, 16), (6, 3, 96, 24), (8, 1, 256, 16), (4, 4, 8, 5),
    (3, 1, 40, 1), (2, 2, 16, 4), (5, 1, 160, 48), (16, 1, 128, 16), (2, 1, 248, 7),
]


# ------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("heads, kv_heads, D, page_size", GEOMETRIES)
def test_attention_over_geometries(ops, workspace, dtype, heads, kv_heads, D, page_size):
    step = Step(dtype, heads, kv_heads, D, page_size, [5, 0, 1, 17, 2], [99, 3, 0, 200, 1], extra_columns=8)
    step.check(step.run(ops, workspace))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("heads, kv_heads, D, page_size", GEOMETRIES)
def test_requests_without_nodes_take_nothing_from_the_scratch(ops, dtype, heads, kv_heads, D, page_size):
    """Whatever the scratch holds where a request without nodes would have its place: here, small numbers that could be blocks' and rows'."""
    from ferrisinfer_b200.engine.workspace import Workspace

    step = Step(dtype, heads, kv_heads, D, page_size, [0, 5, 0, 0, 17, 0], [7, 99, 3, 300, 200, 0])
    for numbers in ([0, 3], [2, 9], [0, 1, 0, 0], [1, 0]):
        workspace = Workspace(DEV)
        workspace.get("tree_attention", (1 << 24,), torch.float32).view(torch.int32).copy_(ints(numbers).repeat((1 << 24) // len(numbers)))
        out = torch.full((22, heads * D), 7.0, dtype=dtype, device=DEV)
        ops.tree_attention(step.q, out, step.k, step.v, ints(step.tables), ints(step.q_start), ints(step.starts), ints(step.parents), *step.most, heads,
                           D ** -0.5, workspace=workspace)
        step.check(out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("kind", ["tree", "chain", "star", "roots"])
@pytest.mark.parametrize("nodes, starts", [([1], [0]), ([1], [1]), ([2], [15]), ([8, 8, 8], [16, 17, 31]), ([33, 64], [128, 127]), ([256, 3], [5, 700]),
                                           ([65], [0]), ([31, 32], [32, 33])])
def test_attention_of_trees(ops, workspace, dtype, kind, nodes, starts):
    step = Step(dtype, 4, 2, 64, 16, nodes, starts, kind)
    step.check(step.run(ops, workspace))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("D", [64, 128, 24])
@pytest.mark.parametrize("window", [1, 2, 7, 33, 100, 4000])
def test_attention_within_a_window(ops, workspace, dtype, D, window):
    step = Step(dtype, 6, 2, D, 16, [12, 30, 1, 9], [400, 40, 7, 0], "chain" if window % 2 else "tree")
    step.check(step.run(ops, workspace, window), window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("seqs, nodes, start, D", [(1, 5, 3000, 64), (1, 64, 1500, 128), (2, 3, 20000, 128), (40, 4, 300, 64)])
def test_attention_over_long_texts(ops, workspace, dtype, seqs, nodes, start, D):
    step = Step(dtype, 4, 1, D, 16, [nodes] * seqs, [start - 7 * i for i in range(seqs)])
    step.check(step.run(ops, workspace))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("D", [64, 128, 32])
def test_rows_without_a_page_are_not_seen(ops, workspace, dtype, D):
    step = Step(dtype, 4, 2, D, 16, [7, 20, 3], [100, 300, 10], holes=[(0, 2), (0, 6), (1, 0), (1, 3), (1, 18), (2, 0)])
    out = step.run(ops, workspace)
    step.check(out)
    assert (out[27:30] == 0).all()  # the last request has no page at all


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("D", [64, 128, 40])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_a_node_does_not_see_has_no_effect(ops, workspace, dtype, D, bad):
    """A sibling's keys and values are not finite: only the nodes below it are not either."""
    step = Step(dtype, 4, 2, D, 16, [20, 20], [70, 500])
    ref, tol = step.expected()
    row = 500 + 3
    page, off = step.tables[1][row // 16], row % 16
    step.v[page, :, off, ::3] = bad
    if bad != bad:
        step.k[page, :, off] = bad
    out = step.run(ops, workspace)
    lines = plain.lines_of(step.parents[20:])
    sees = torch.tensor([False] * 20 + [3 in line for line in lines])
    step.compare(out, ref, tol, ~sees)
    assert not torch.isfinite(out.cpu()[sees].view(-1, 4, D)[:, :, ::3].float()).any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_before_the_window_have_no_effect(ops, workspace, dtype, D):
    step = Step(dtype, 4, 2, D, 16, [20], [300], "chain")
    ref, tol = step.expected(50)
    for row in range(300 - 50 + 1):
        step.v[step.tables[0][row // 16], :, row % 16] = math.nan
    step.compare(step.run(ops, workspace, 50), ref, tol)
    row = 300 - 50 + 2  # the first that the first node sees is the one before; the second node does not see this one
    step.v[step.tables[0][row // 16], :, row % 16] = math.nan
    out = step.run(ops, workspace, 50)
    assert torch.isnan(out[:2]).all()
    step.compare(out, ref, tol, slice(2, None))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_rows_behind_the_last_request_stay(ops, workspace, dtype):
    step = Step(dtype, 4, 2, 64, 16, [3, 5], [20, 2000], spare_rows=6)
    out = step.run(ops, workspace)
    step.check(out)
    assert (out[8:] == 7).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("D, nodes, start", [(64, 4, 900), (128, 40, 900), (64, 70, 40)])
def test_rows_of_other_matrices(ops, workspace, dtype, D, nodes, start):
    """Queries and outputs as columns of wider matrices, off 16 bytes."""
    step = Step(dtype, 4, 2, D, 16, [nodes, 2], [start, 33])
    whole = step.run(ops, workspace).clone()
    wide = torch.zeros(nodes + 2, 4 * D + 11, dtype=dtype, device=DEV)
    wide[:, 3:3 + 4 * D] = step.q
    step.q = wide[:, 3:]
    out = torch.full((nodes + 2, 4 * D + 5), 7.0, dtype=dtype, device=DEV)
    step.run(ops, workspace, out=out[:, 1:1 + 4 * D])
    assert torch.equal(out[:, 1:1 + 4 * D], whole) and (out[:, 0] == 7).all() and (out[:, 1 + 4 * D:] == 7).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_bounds_of_the_call(ops, workspace, dtype):
    step = Step(dtype, 4, 2, 64, 16, [6, 4], [90, 500])
    out = step.run(ops, workspace, most=(6, 300))  # rows from 300 on are not seen
    step.check(out, max_rows=300)
    out = step.run(ops, workspace, most=(200, 1 << 30))  # far above what there is
    step.check(out)
    out = step.run(ops, workspace, most=(4, 504))  # the first request brings more nodes
    reported(ops, 110)
    ref, _, _ = plain.tree_attention(step.q, step.k, step.v, step.tables, step.q_start, step.starts, step.parents, 4, 0.125, max_nodes=4)
    assert (out[4:6] == 7).all() and torch.allclose(out[:4].double().cpu(), ref[:4], atol=0.05) and torch.allclose(out[6:].double().cpu(), ref[6:], atol=0.05)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_indices_that_cannot_be_are_reported(ops, workspace, dtype):
    step = Step(dtype, 4, 2, 64, 16, [6, 4], [90, 500])
    step.parents[3], step.parents[7] = 3, -2  # itself; below -1: both count as none
    out = step.run(ops, workspace)
    reported(ops, 112)
    step.check(out)
    step = Step(dtype, 4, 2, 64, 16, [6, 4], [90, 500])
    step.tables[1][2] = step.k.shape[0]  # no such page
    out = step.run(ops, workspace)
    reported(ops, 111)
    step.tables[1][2] = -1
    step.check(out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_the_same_bits_from_run_to_run_on_other_streams_and_recorded(ops, dtype):
    from ferrisinfer_b200.engine.workspace import Workspace

    workspace = Workspace(DEV)
    steps = [Step(dtype, 14, 2, 64, 16, [9] * 6, [1700] * 6, seed=3), Step(dtype, 14, 2, 64, 16, [40], [5000], seed=4)]
    want = [step.run(ops, workspace).clone() for step in steps]
    for step, out in zip(steps, want):
        assert torch.equal(step.run(ops, workspace), out)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = [step.run(ops, workspace) for step in steps]
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # two recorded steps that share the workspace, replayed one after the other
    outs, graphs = [torch.zeros_like(x) for x in want], []
    workspace.pin()
    for step, out in zip(steps, outs):
        tensors = step.device_tensors
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.tree_attention(step.q, out, step.k, step.v, *tensors, *step.most, step.heads, step.D ** -0.5, workspace=workspace)
        graphs.append(graph)
    for _ in range(3):
        for graph, out in zip(graphs, outs):
            out.zero_()
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_offsets_beyond_32_bits(ops, workspace):
    """A cache of more than 2^31 elements, of whose last pages a request has some."""
    pages, hkv, ps, D = (1 << 31) // (2 * 16 * 128) + 64, 2, 16, 128
    if torch.cuda.mem_get_info()[0] < 5 * pages * hkv * ps * D:
        pytest.skip("not enough memory")
    k, v = (torch.empty(pages, hkv, ps, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    gen = rng(5)
    table = [pages - 1 - i for i in range(20)]
    for t in (k, v):
        t[pages - 20:] = torch.randn(20, hkv, ps, D, generator=gen, device=DEV).to(torch.bfloat16)
    for n in (3, 40):
        q = torch.randn(n, 4 * D, generator=gen, device=DEV).to(torch.bfloat16)
        out, parents = torch.zeros_like(q), tree(n, "tree")
        ops.tree_attention(q, out, k, v, ints([table]), ints([0, n]), ints([270]), ints(parents), n, 320, 4, 0.09, workspace=workspace)
        ref, mag, size = plain.tree_attention(q, k, v, [table], [0, n], [270], parents, 4, 0.09)
        assert ((out.double().cpu() - ref).abs() <= plain.attention_tolerance(torch.bfloat16, ref, mag, size, 310, D)).all()


# ------------------------------------------------------------------------------------------------ probabilities
def check_probs(ops, logits, temperature, top_k, top_p, out=None):
    n = logits.shape[0]
    as_list = lambda x: list(x) if isinstance(x, (list, tuple)) else [x] * n
    temperature, top_p = (torch.tensor(as_list(x), dtype=torch.float32) for x in (temperature, top_p))
    top_k = as_list(top_k)
    out = torch.full(logits.shape, 9.0, device=DEV) if out is None else out
    ref = plain.sampling_probs(logits, temperature.tolist(), top_k, top_p.tolist())
    ops.sampling_probs(logits, out, temperature.to(DEV), ints(top_k), top_p.to(DEV))
    got = out.double().cpu()
    assert torch.equal(got > 1e-30, ref > 1e-30)
    # an exponent (l - max) / T of 32 bits is off by 2^-23 of itself, the exponential, the sum and the quotient by a few 2^-24
    finite = torch.where(torch.isfinite(logits), logits, 0.0).double().cpu()
    exponent = ((finite.amax(1, keepdim=True) - finite) / temperature.double()[:, None].clamp(min=1e-6)).abs().clamp(max=104.0)
    assert ((got - ref).abs() <= ref * (exponent * 2.0 ** -22 + 2.0 ** -19) + 1e-37).all()
    return out


def logits_of(n, V, seed=0):
    return torch.randn(n, V, generator=rng(seed + V), device=DEV) * 3


@pytest.mark.parametrize("V", [1, 2, 3, 31, 257, 1000, 4099, 32003])
@pytest.mark.parametrize("temperature, top_k, top_p", [(1.0, 0, 1.0), (0.7, 20, 0.9), (0.8, 0, 0.9), (1.3, 7, 1.0), (0.0, 5, 0.5), (0.5, 1, 1.0), (0.6, 600, 0.97),
                                                       (1.0, 5, 0.0), (2.0, 100000, 0.3), (1.0, 0, 1e-6), (0.9, 3, 0.999999)])
def test_probabilities(ops, V, temperature, top_k, top_p):
    check_probs(ops, logits_of(3, V), temperature, top_k, top_p)


def test_probabilities_of_rows_with_options_of_their_own(ops):
    check_probs(ops, logits_of(7, 5003), [0.0, 1.0, 0.7, 0.5, 1e-9, 3.0, 0.01], [1, 0, 20, 900, 4, 2, 0], [1.0, 1.0, 0.9, 0.8, 1.0, 1.0, 0.5])


@pytest.mark.parametrize("V", [7, 1030, 4099])
def test_probabilities_of_many_rows(ops, V):
    """(more than run at once, plain ones among others)"""
    n = 150
    logits = logits_of(n, V)
    logits[3], logits[4], logits[5, ::2], logits[6], logits[7] = -math.inf, math.nan, math.nan, 2.5, -math.inf
    logits[7, V // 2], logits[8, 5], logits[9, V - 1] = 1.0, math.inf, -math.inf
    options = [(1.0, 0, 1.0), (0.7, 5, 0.9), (0.5, 0, 1.0), (0.0, 0, 1.0), (1.0, 0, 0.8), (2.0, V, 1.0), (1.0, 1, 1.0)]
    for first in ([(1.0, 0, 1.0)] * n, [options[i % 7] for i in range(n)], [options[1]] * n):
        check_probs(ops, logits, *zip(*first))
    wide = torch.zeros(n, V + 9, device=DEV)
    wide[:, 3:3 + V] = logits
    want, out = torch.empty_like(logits), torch.full((n, V + 6), 9.0, device=DEV)
    ops.sampling_probs(logits, want, torch.ones(n, device=DEV))
    ops.sampling_probs(wide[:, 3:3 + V], out[:, 1:1 + V], torch.ones(n, device=DEV))
    assert torch.allclose(out[:, 1:1 + V], want, rtol=1e-5, atol=1e-37) and (out[:, 0] == 9).all() and (out[:, 1 + V:] == 9).all()
    same = logits.clone()
    ops.sampling_probs(same, same, torch.ones(n, device=DEV))
    assert torch.equal(same, want)


@pytest.mark.parametrize("V", [11, 2048, 20001])
@pytest.mark.parametrize("top_k, top_p", [(0, 0.5), (5, 1.0), (700, 1.0), (700, 0.25), (0, 1.0), (10, 0.5), (0, 0.125)])
def test_equal_logits_stay_by_their_index(ops, V, top_k, top_p):
    logits = torch.zeros(4, V, device=DEV)
    logits[1] = -0.0
    logits[1, ::2] = 0.0  # the two noughts are one
    logits[2, V // 2:] = 1.0
    logits[3] = (torch.arange(V, device=DEV) % 3).float()
    check_probs(ops, logits, 1.0, top_k, top_p)


@pytest.mark.parametrize("top_k, top_p", [(0, 1.0), (3, 1.0), (0, 0.6), (3, 0.6), (600, 0.9), (1, 1.0)])
def test_logits_that_are_not_finite(ops, top_k, top_p):
    inf, nan = math.inf, math.nan
    logits = logits_of(8, 1500)
    logits[0, ::2] = -inf
    logits[1] = -inf
    logits[2] = nan
    logits[3, 5:] = nan
    logits[4, 77] = inf
    logits[5, 100:900] = inf
    logits[6] = -inf
    logits[6, 1400] = 3.0
    logits[7, 1::2] = torch.finfo(torch.float32).min
    check_probs(ops, logits, 0.8, top_k, top_p)


@pytest.mark.parametrize("spread", [1e-4, 1e-30, 1e4, 1e36])
@pytest.mark.parametrize("temperature", [1e-4, 1.0, 1e5])
@pytest.mark.parametrize("top_k, top_p", [(600, 0.9), (40, 0.7), (0, 0.7), (0, 1.0)])
def test_logits_of_any_spread(ops, spread, temperature, top_k, top_p):
    logits = torch.randn(2, 6007, generator=rng(8), device=DEV).double()
    check_probs(ops, (logits * spread).float(), temperature, top_k, top_p)


def test_a_cluster_of_logits_beside_far_ones(ops):
    """All but a few logits fall into one bin of any histogram over the row's range."""
    logits = 1e-3 * torch.randn(2, 9001, generator=rng(9), device=DEV)
    logits[:, :3] = torch.tensor([1e6, -1e6, 5e5], device=DEV)
    for temperature, top_k, top_p in ((1e6, 5000, 1.0), (1e6, 0, 0.5), (1e6, 800, 0.9), (1e6, 10, 0.9)):
        check_probs(ops, logits, temperature, top_k, top_p)


def test_probabilities_in_place_and_of_rows_of_other_matrices(ops):
    logits = logits_of(5, 3001)
    want = check_probs(ops, logits, 0.8, 40, 0.9)
    check_probs(ops, logits.clone(), 0.8, 40, 0.9, out=None)
    same = logits.clone()
    ops.sampling_probs(same, same, torch.full((5,), 0.8, device=DEV), ints([40] * 5), torch.full((5,), 0.9, device=DEV))
    assert torch.equal(same, want)
    wide, other = torch.zeros(5, 3011, device=DEV), torch.full((5, 3010), 9.0, device=DEV)
    wide[:, 3:3004] = logits
    ops.sampling_probs(wide[:, 3:3004], other[:, 1:3002], torch.full((5,), 0.8, device=DEV), ints([40] * 5), torch.full((5,), 0.9, device=DEV))
    assert torch.equal(other[:, 1:3002], want) and (other[:, 0] == 9).all() and (other[:, 3002:] == 9).all()
    shared = logits[:1].expand(5, 3001)
    out = torch.zeros(5, 3001, device=DEV)
    ops.sampling_probs(shared, out, torch.full((5,), 0.8, device=DEV), ints([40] * 5), torch.full((5,), 0.9, device=DEV))
    assert all(torch.equal(out[i], want[0]) for i in range(5))


def test_options_left_out(ops):
    logits = logits_of(2, 700)
    out = torch.empty_like(logits)
    ops.sampling_probs(logits, out)
    assert torch.equal(out, torch.nn.functional.one_hot(logits.argmax(1), 700).float())
    ops.sampling_probs(logits, out, torch.ones(2, device=DEV))
    assert torch.allclose(out.double(), torch.softmax(logits.double(), 1), rtol=1e-5)


@pytest.mark.parametrize("V", [151936, 500003])
def test_large_vocabularies(ops, V):
    """(the second one's rows do not fit the shared memory of a row's blocks)"""
    logits = logits_of(4, V)
    out = torch.empty_like(logits)
    for T, k, p in ((1.0, 0, 1.0), (0.7, 20, 0.9), (0.9, 0, 0.95), (1.0, 3001, 0.9)):
        ops.sampling_probs(logits, out, torch.full((4,), T, device=DEV), ints([k] * 4), torch.full((4,), p, device=DEV))
        x = logits.double()
        w, order = torch.sort(torch.exp((x - x.amax(1, keepdim=True)) / T), dim=1, descending=True, stable=True)
        w = torch.where((torch.arange(V, device=DEV) < k) if k else torch.ones(V, dtype=torch.bool, device=DEV), w, 0.0)
        if p < 1:
            w = torch.where(torch.cumsum(w, 1) - w < torch.tensor(p, dtype=torch.float32).item() * w.sum(1, keepdim=True), w, 0.0)
        ref = torch.zeros_like(x).scatter_(1, order, w / w.sum(1, keepdim=True))
        assert torch.equal(out > 0, ref.float() > 0) and torch.allclose(out.double(), ref, rtol=2e-5, atol=1e-37)
        first = out.clone()
        ops.sampling_probs(logits, out, torch.full((4,), T, device=DEV), ints([k] * 4), torch.full((4,), p, device=DEV))
        assert torch.equal(first, out)


def test_probabilities_are_those_that_the_sampler_draws_by(ops):
    """Tokens of many draws come as often as the probabilities say."""
    n, V = 20000, 60
    row = torch.randn(1, V, generator=rng(12), device=DEV) * 2
    probs = torch.empty_like(row)
    ops.sampling_probs(row, probs, torch.tensor([0.8], device=DEV), ints([20]), torch.tensor([0.9], device=DEV))
    tokens, states = torch.empty(n, dtype=torch.int32, device=DEV), torch.arange(1, n + 1, dtype=torch.int64, device=DEV) * 0x1E3779B97F4A7C15 % (1 << 62)
    ops.sample(row.expand(n, V).contiguous(), tokens, None, torch.full((n,), 0.8, device=DEV), ints([20] * n), torch.full((n,), 0.9, device=DEV),
               torch.arange(n, dtype=torch.int32, device=DEV), states)
    count = torch.bincount(tokens.long(), minlength=V).double()
    p = probs[0].double()
    assert (count[p == 0] == 0).all()
    # (six standard deviations and one draw)
    assert ((count - n * p).abs() <= 6 * (n * p * (1 - p)).sqrt() + 1).all()


# ------------------------------------------------------------------------------------------------ verification
def run_verify(ops, probs, tokens, parents, q_start, uniforms, width, draft=None):
    S = len(q_start) - 1
    nodes, accepted, token = (torch.full(shape, -9, dtype=torch.int32, device=DEV) for shape in ((S, width), (S,), (S,)))
    ops.verify_tree(probs, ints(tokens), ints(parents), ints(q_start), torch.tensor(uniforms, dtype=torch.float32, device=DEV), nodes, accepted, token,
                    draft_probs=draft)
    return nodes.tolist(), accepted.tolist(), token.tolist()


def check_verify(ops, probs, tokens, parents, q_start, uniforms, width, draft=None):
    uniforms = torch.tensor(uniforms, dtype=torch.float32).tolist()
    got = run_verify(ops, probs, tokens, parents, q_start, uniforms, width, draft)
    assert got == plain.verify_tree(probs, tokens, parents, q_start, uniforms, width, draft)
    return got


def drafted_step(V, nodes, kind, drafted, seed, sharp=2.0):
    gen, draw = rng(seed), random.Random(seed)
    T = sum(nodes)
    base = torch.randn(T, V, generator=gen, device=DEV) * sharp
    draft = torch.softmax(base, 1) if drafted else None
    probs = torch.softmax(base + 0.6 * torch.randn(T, V, generator=gen, device=DEV), 1)
    q_start, parents, tokens = [0], [], []
    for i, n in enumerate(nodes):
        parents += tree(n, kind, seed + i)
        q_start.append(q_start[-1] + n)
    source = (draft if drafted else probs).cpu()
    for first, n in zip(q_start, nodes):
        for c in range(n):
            row = source[first + max(parents[first + c], 0)]
            tokens.append(int(torch.searchsorted(torch.cumsum(row, 0), torch.tensor(draw.random()))) % V)
    return probs, tokens, parents, q_start, [draw.random() for _ in range(T)], draft


@pytest.mark.parametrize("drafted", [False, True], ids=["chosen", "drawn"])
@pytest.mark.parametrize("kind", ["chain", "tree", "star", "roots"])
@pytest.mark.parametrize("V", [1, 2, 5, 130, 1001, 32003])
def test_verification(ops, drafted, kind, V):
    for seed in range(3):
        probs, tokens, parents, q_start, u, draft = drafted_step(V, [1, 5, 0, 17, 2, 9], kind, drafted, seed)
        check_verify(ops, probs, tokens, parents, q_start, u, 17, draft)


@pytest.mark.parametrize("drafted", [False, True], ids=["chosen", "drawn"])
def test_verification_of_a_large_vocabulary(ops, drafted):
    probs, tokens, parents, q_start, u, draft = drafted_step(151936, [8] * 6, "tree", drafted, 5, sharp=3.0)
    first = check_verify(ops, probs, tokens, parents, q_start, u, 8, draft)
    assert run_verify(ops, probs, tokens, parents, q_start, u, 8, draft) == first


@pytest.mark.parametrize("drafted", [False, True], ids=["chosen", "drawn"])
def test_large_trees_and_short_paths(ops, drafted):
    probs, tokens, parents, q_start, u, draft = drafted_step(40, [256, 3, 100], "tree", drafted, 6)
    check_verify(ops, probs, tokens, parents, q_start, u, 256, draft)
    u = [0.0] * len(u)  # everything that can be is accepted; paths end where they are full
    for width in (1, 2, 4):
        _, accepted, _ = check_verify(ops, probs, tokens, parents, q_start, u, width, draft)
        assert max(accepted) == width - 1
    probs, tokens, parents, q_start, u, draft = drafted_step(300, [256], "star", drafted, 7)
    check_verify(ops, probs, tokens, parents, q_start, [0.999] * 256, 256, draft)  # nearly everything is refused


@pytest.mark.parametrize("drafted", [False, True], ids=["chosen", "drawn"])
def test_random_numbers_at_the_ends(ops, drafted):
    probs, tokens, parents, q_start, u, draft = drafted_step(1001, [4] * 3, "star", drafted, 8)
    tops = 1 - 2.0 ** -24
    for value in (0.0, tops):
        check_verify(ops, probs, tokens, parents, q_start, [value] * 12, 4, draft)
    check_verify(ops, probs, tokens, parents, q_start, [tops, 0.5, 0.0, tops] * 3, 4, draft)


def test_rows_of_one_token_and_of_none(ops):
    V = 70
    probs = torch.zeros(12, V, device=DEV)
    probs[:4, 7] = 1.0  # greedy rows
    probs[4:8, 69] = 1.0
    check_verify(ops, probs, [3, 7, 7, 8] + [1, 69, 0, 69] + [0, 1, 2, 3], [-1, 0, 0, 1] + [-1, 0, 1, 2] + [-1, 0, 1, 2], [0, 4, 8, 12], [0.5] * 12, 4)
    got = run_verify(ops, probs, [3, 7, 7, 8] + [1, 69, 0, 69] + [0, 1, 2, 3], [-1, 0, 0, 1] + [-1, 0, 1, 2] + [-1, 0, 1, 2], [0, 4, 8, 12], [0.5] * 12, 4)
    assert got == ([[0, 1, -1, -1], [0, 1, -1, -1], [0, -1, -1, -1]], [1, 1, 0], [7, 69, -1])


def test_siblings_of_one_token_and_drafts_that_know_the_target(ops):
    V = 9
    probs = torch.softmax(torch.randn(4, V, generator=rng(3), device=DEV), 1)
    # the same token three times: refused once, it has no probability left
    for u in (0.0, 0.3, 0.9):
        check_verify(ops, probs, [0, 4, 4, 4], [-1, 0, 0, 0], [0, 4], [u, 0.99, 0.0, 0.0], 4)
        # a draft that is the target: the residual is nothing, the target's row stays
        check_verify(ops, probs, [0, 4, 4, 2], [-1, 0, 0, 0], [0, 4], [u, 1 - 2.0 ** -24, 0.5, 0.5], 4, probs.clone())
    draft = probs.clone()
    draft[:, 4] = 0  # a token that the draft says it cannot have drawn
    check_verify(ops, probs, [0, 4, 4, 2], [-1, 0, 0, 0], [0, 4], [0.5, 0.99, 0.5, 0.5], 4, draft)


def test_values_that_are_no_probabilities(ops):
    probs, tokens, parents, q_start, u, draft = drafted_step(50, [6, 6], "tree", True, 9)
    probs[:, ::5] = math.nan
    probs[:, 1::5] = -0.5
    draft[:, 2::5] = math.nan
    for d in (None, draft):
        check_verify(ops, probs, tokens, parents, q_start, u, 6, d)


def test_verification_of_rows_of_other_matrices(ops):
    probs, tokens, parents, q_start, u, draft = drafted_step(1003, [6, 6], "tree", True, 10)
    want = check_verify(ops, probs, tokens, parents, q_start, u, 6, draft)
    wide = torch.full((2, 12, 1010), math.nan, device=DEV)
    wide[0, :, 3:1006], wide[1, :, 1:1004] = probs, draft
    assert run_verify(ops, wide[0, :, 3:1006], tokens, parents, q_start, u, 6, wide[1, :, 1:1004]) == want


def test_verification_reports_what_cannot_be(ops):
    probs, tokens, parents, q_start, u, _ = drafted_step(30, [5, 5], "chain", False, 11)
    u = [0.0] * 10
    tokens[7] = 30
    check_verify(ops, probs, tokens, parents, q_start, u, 5)
    reported(ops, 132)
    tokens[7] = -1
    check_verify(ops, probs, tokens, parents, q_start, u, 5)
    reported(ops, 132)
    tokens[7], parents[3] = 3, 4
    check_verify(ops, probs, tokens, parents, q_start, u, 5)
    reported(ops, 131)
    probs, tokens, parents, q_start, u, _ = drafted_step(30, [300], "tree", False, 12)
    check_verify(ops, probs, tokens, parents, q_start, u, 300)
    reported(ops, 130)


@pytest.mark.parametrize("drafted", [False, True], ids=["chosen", "drawn"])
def test_tokens_follow_the_target(ops, drafted):
    """Over many requests of one tree, the first token that comes out is distributed as the target's row, whatever was drafted."""
    V, S, gen, draw = 6, 30000, rng(21), random.Random(4)
    p = torch.softmax(torch.randn(V, generator=gen, device=DEV), 0)
    q = torch.softmax(torch.randn(V, generator=gen, device=DEV), 0)
    n = 4  # the known token and three children
    probs = p.expand(S * n, V).contiguous()
    cum = torch.cumsum(q.double(), 0).cpu()
    drawn = torch.searchsorted(cum, torch.rand(S, n, generator=gen, device=DEV).double().cpu() * cum[-1]).clamp(max=V - 1)
    tokens = drawn if drafted else torch.tensor([0, 2, 5, 2]).expand(S, n)
    u = torch.rand(S * n, generator=gen, device=DEV)
    nodes, accepted, token = (torch.zeros(shape, dtype=torch.int32, device=DEV) for shape in ((S, 2), (S,), (S,)))
    ops.verify_tree(probs, tokens.reshape(-1).to(torch.int32).to(DEV), ints([-1, 0, 0, 0]).repeat(S), ints(range(0, S * n + 1, n)), u, nodes, accepted, token,
                    draft_probs=q.expand(S * n, V).contiguous() if drafted else None)
    first = torch.where(accepted.cpu() > 0, tokens[torch.arange(S), nodes[:, 1].cpu().clamp(min=0).long()].to(torch.int32), token.cpu())
    count, want = torch.bincount(first.long(), minlength=V).double(), S * p.double().cpu()
    assert ((count - want).abs() <= 6 * (want * (1 - want / S)).sqrt()).all()
    assert accepted.float().mean() > 0.1


# ------------------------------------------------------------------------------------------------ rows kept
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16], ids=["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("layers, kv_heads, D, page_size", [(1, 1, 64, 16), (3, 2, 128, 16), (2, 3, 20, 5), (2, 1, 7, 1), (5, 4, 96, 64)])
def test_rows_of_the_accepted_nodes_move(ops, dtype, layers, kv_heads, D, page_size):
    if dtype == torch.float32 and D == 7:
        page_size = 3
    starts = [0, 1, 15, 100, 37, 64, 9]
    nodes = [[0, 1, 2, 3, -1, -1], [0, 2, 3, 5, 9, 10], [0, 5, -1, -1, -1, -1], [0, -1, -1, -1, -1, -1], [0, 3, 4, 5, 11, 12], [0, 2, 4, 5, -1, -1], [0, 1, 3, 4, 6, 7]]
    accepted = [3, 5, 1, 0, 5, 2, 9]  # (fewer than the path has; more than it has room for)
    blocks = [-(-(s + 13) // page_size) for s in starts]
    order, at, tables = random.Random(1).sample(range(sum(blocks) + 2), sum(blocks) + 2), 0, []
    for b in blocks:
        tables.append(order[at:at + b] + [-1] * (max(blocks) - b))
        at += b
    gen = rng(2)
    caches = [[torch.randn(len(order), kv_heads, page_size, D, generator=gen, device=DEV).to(dtype) for _ in range(2)] for _ in range(layers)]
    want = [t.cpu() for layer in caches for t in layer]
    plain.keep_tree_rows(want, tables, starts, nodes, accepted)
    handle = ops.CacheLayers(caches)
    ops.keep_tree_rows(handle, ints(tables), ints(starts), ints(nodes), ints(accepted))
    assert all(torch.equal(a.cpu(), b) for a, b in zip([t for layer in caches for t in layer], want))


def test_long_paths_move(ops):
    n = 256
    for path in ([0] + list(range(2, 129)), list(range(256)), [0] + list(range(100, 255))):
        cache = torch.randn(2, 30, 1, 16, 8, device=DEV)
        table, start = random.Random(3).sample(range(30), 30), 77
        want = [cache[0].cpu(), cache[1].cpu()]
        nodes = path + [-1] * (n - len(path))
        plain.keep_tree_rows(want, [table], [start], [nodes], [len(path) - 1])
        ops.keep_tree_rows(ops.CacheLayers([(cache[0], cache[1])]), ints([table]), ints([start]), ints([nodes]), ints([len(path) - 1]))
        assert torch.equal(cache[0].cpu(), want[0]) and torch.equal(cache[1].cpu(), want[1])


def test_moves_that_cannot_be_are_reported(ops):
    cache = torch.randn(2, 8, 1, 4, 8, device=DEV)
    handle, before = ops.CacheLayers([(cache[0], cache[1])]), cache.clone()
    tables = [list(range(8))]
    for nodes, moved in (([0, 3, 3, 6], 1), ([0, 3, 5, 2], 2), ([0, 0, 5, 6], 0), ([0, -1, 5, 6], 0)):
        cache.copy_(before)
        want = [before[0].cpu(), before[1].cpu()]
        plain.keep_tree_rows(want, tables, [4], [nodes], [moved])
        ops.keep_tree_rows(handle, ints(tables), ints([4]), ints([nodes]), ints([3]))
        reported(ops, 120)
        assert torch.equal(cache[0].cpu(), want[0]) and torch.equal(cache[1].cpu(), want[1])
    # rows without a page, and such as no table names
    for table, nodes in (([0, 1, 2, -1] + [4] * 4, [0, 9, 10, 11]), ([0, 1, 2, 8] + [4] * 4, [0, 9, 10, 11]), (list(range(8)), [0, 29, 30, 1 << 30])):
        cache.copy_(before)
        ops.keep_tree_rows(handle, ints([table]), ints([4]), ints([nodes]), ints([3]))
        reported(ops, 121)
    cache.copy_(before)
    ops.keep_tree_rows(handle, ints(tables), ints([-1]), ints([[0, 2, 3]]), ints([2]))
    ops.keep_tree_rows(handle, ints(tables), ints([3]), ints([[0, 2, 3]]), ints([-5]))
    assert torch.equal(cache, before)


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals(ops, workspace):
    from ferrisinfer_b200.errors import KernelError

    step = Step(torch.bfloat16, 4, 2, 64, 16, [3, 2], [20, 30])
    step.run(ops, workspace)
    tables, q_start, starts, parents = step.device_tensors
    out = torch.zeros(5, 256, dtype=torch.bfloat16, device=DEV)
    good = dict(q=step.q, out=out, k_cache=step.k, v_cache=step.v, block_tables=tables, seq_q_start=q_start, seq_start_row=starts, parents=parents,
                max_q_len=3, max_kv_len=40, num_heads=4, scale=0.125, workspace=workspace)
    ops.tree_attention(**good)
    wide = torch.zeros(3, 2, 16, 264, dtype=torch.bfloat16, device=DEV)
    for change, words in ((dict(q=step.q.cpu()), "one device"), (dict(q=step.q.float()), "all float32 or all bfloat16"), (dict(parents=parents.long()), "int32"),
                          (dict(block_tables=tables[:, ::2]), "contiguous"), (dict(num_heads=3), "cannot share"), (dict(max_q_len=257), "256"),
                          (dict(window=-1), "window"), (dict(parents=parents[:4]), "parents"), (dict(q=step.q.T), "q "), (dict(workspace=None), "workspace"),
                          (dict(k_cache=step.k[:, :, :8]), "contiguous"), (dict(seq_q_start=q_start[:2]), "first rows"), (dict(out=out[:, ::2]), "out"),
                          (dict(k_cache=wide, v_cache=wide, q=torch.zeros(5, 4 * 264, dtype=torch.bfloat16, device=DEV),
                                out=torch.zeros(5, 4 * 264, dtype=torch.bfloat16, device=DEV)), "at most 256"),
                          (dict(max_kv_len=0), "no rows")):
        with pytest.raises(KernelError, match=words):
            ops.tree_attention(**{**good, **change})
    logits, flat = torch.zeros(4, 100, device=DEV), torch.zeros(1000, device=DEV)
    with pytest.raises(KernelError, match="float32"):
        ops.sampling_probs(logits.half(), logits)
    with pytest.raises(KernelError, match="apart"):
        ops.sampling_probs(flat[:400].view(4, 100), flat[10:410].view(4, 100))
    with pytest.raises(KernelError, match="overlap"):
        ops.sampling_probs(logits, flat[:100].expand(4, 100))
    with pytest.raises(KernelError, match="524288"):
        ops.sampling_probs(torch.zeros(1, 524289, device=DEV), torch.zeros(1, 524289, device=DEV))
    with pytest.raises(KernelError, match="top_k"):
        ops.sampling_probs(logits, torch.zeros_like(logits), torch.ones(4, device=DEV), torch.ones(4, device=DEV))
    with pytest.raises(KernelError, match="one device"):
        ops.sampling_probs(logits.cpu(), logits)
    probs, one = torch.zeros(5, 30, device=DEV), ints([0, 5])
    i5, nodes, s1 = ints([0] * 5), ints([[0, 0]]), ints([0])
    good = dict(probs=probs, tokens=i5, parents=i5, seq_q_start=one, uniforms=torch.zeros(5, device=DEV), out_nodes=nodes, out_accepted=s1, out_token=s1.clone())
    ops.verify_tree(**good)
    for change, words in ((dict(tokens=i5[:3]), "tokens"), (dict(uniforms=torch.zeros(5, device=DEV, dtype=torch.float64)), "random numbers"),
                          (dict(out_nodes=ints([0])), "paths"), (dict(draft_probs=probs[:4]), "draft"), (dict(probs=probs.T), "probabilities"),
                          (dict(tokens=i5.long()), "int32"), (dict(parents=i5.cpu()), "one device")):
        with pytest.raises(KernelError, match=words):
            ops.verify_tree(**{**good, **change})
    cache = torch.zeros(4, 2, 16, 8, device=DEV)
    layers = ops.CacheLayers([(cache, cache.clone())])
    table = ints([[0, 1]])
    ops.keep_tree_rows(layers, table, s1, nodes, s1)
    with pytest.raises(KernelError, match="CacheLayers"):
        ops.keep_tree_rows([(cache, cache)], table, s1, nodes, s1)
    with pytest.raises(KernelError, match="at most 256"):
        ops.keep_tree_rows(layers, table, s1, torch.zeros(1, 257, dtype=torch.int32, device=DEV), s1)
    with pytest.raises(KernelError, match="requests"):
        ops.keep_tree_rows(layers, table, s1, nodes, ints([0, 0]))
    with pytest.raises(KernelError, match="none are given"):
        ops.CacheLayers([])
    with pytest.raises(KernelError, match="beside"):
        ops.CacheLayers([(cache, cache[:2])])
    with pytest.raises(KernelError, match="contiguous"):
        ops.CacheLayers([(cache[:, :, ::2], cache[:, :, ::2])])
