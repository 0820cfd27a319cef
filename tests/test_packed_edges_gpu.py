"""The packed cache at its edges: values far apart, rows and scores that are no numbers, loose bounds, holes, slots."""

import math

import pytest
import torch

import plain_packed as plain
from test_packed_cache_gpu import make_step, packed

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from ferrisinfer_b200.kernels import ops as module

    module.require_device()
    return module


@pytest.fixture(autouse=True)
def no_wait_ran_out(ops):
    yield
    torch.cuda.synchronize()
    ops.check_kernel_status()


@pytest.fixture(scope="module")
def workspace():
    from ferrisinfer_b200.engine.workspace import Workspace

    return Workspace(DEV)


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def parts_of(cache, table, rows, page_size):
    """|middle| + 8 scale of every element of the values of a request's rows, 64 bits: what stands in its sums beside what
    the two make together (a value is middle + scale x (code - 8))."""
    r = torch.arange(rows, device=DEV)
    page = table.long()[(r // page_size).clamp(max=table.numel() - 1)].clamp(min=0)
    s = cache[3][page, :, r % page_size].double()
    return ((s[..., 1] + 8 * s[..., 0]).abs() + 8 * s[..., 0]).repeat_interleave(32, -1)


def attend_and_compare(ops, workspace, step, lengths, heads, kv_heads, D, page_size, scale=None, window=0, max_q=None, max_kv=None, far=()):
    """One step with the rows' weights against the plain form; the bounds follow each number's own sums.  ``far``: (request, row) whose
    weight is nought whatever the last bits of its score."""
    cache, tables, q, q_start, start_row, rows = step
    scale = D ** -0.5 if scale is None else scale
    most = max(rows)
    out = torch.full((q.shape[0], heads * D), 7.0, dtype=q.dtype, device=DEV)
    weights = torch.full((len(lengths), kv_heads, most), 3.0, device=DEV)
    ops.packed_attention(q, out, packed(ops, cache), tables, q_start, start_row, max(n for n, _ in lengths) if max_q is None else max_q,
                         most if max_kv is None else max_kv, heads, scale, window=window,
                         weights=weights if max_kv is None else None, add_weights=False, workspace=workspace)
    at = 0
    for i, ((n, start), r) in enumerate(zip(lengths, rows)):
        k, v, has = plain.request_rows(cache, tables[i], r, page_size)
        mine = q[at:at + n].double().view(n, heads, D)
        want, w, _, _ = plain.attend(mine, k, v, has, start, scale, window)
        near = has.clone()
        near[[row for request, row in far if request == i]] = False
        spread = plain.attend(mine, k, v, near, start, scale, window)[3]
        size = plain.attend(mine, k, parts_of(cache, tables[i], r, page_size), has, start, scale, window)[0]
        # Scores: a sum of D / 8 + 8 steps of 24-bit numbers (cut rather than rounded), twice: in a weight and in the sum that it is
        # divided by; the exponential and the weights' sums beside them.  Outputs: for bf16 rows weights, and their products
        # with scales, in eleven bits (2^-9 covers both and their sum), and the result once more; else 24-bit sums.
        rel = (D / 8 + 8) * 2.0 ** -23 * spread * 2 + 2.0 ** -19
        lossy = 2.0 ** -9 if q.dtype == torch.bfloat16 else 0.0
        bound = size * (rel[..., None] + lossy) + want.abs() * (lossy + 2.0 ** -23) + 1e-30
        got = out[at:at + n].double().view(n, heads, D)
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(got), nan), (i, (torch.isnan(got) != nan).nonzero()[:4])
        assert ((got - want).abs() <= bound)[~nan].all(), (i, ((got - want).abs() / bound)[~nan].max())
        if max_kv is None and n:
            g, nan = weights[i, :, :r].double(), torch.isnan(w)
            assert torch.equal(torch.isnan(g), nan)
            e = rel.nan_to_num(0.0).max()
            assert ((g - w).abs() <= w * (e + 2.0 ** -20) + 1e-30)[~nan].all(), (i, ((g - w).abs() / (w * e + 1e-30))[~nan].max())
        at += n
    return out


def with_queries(step, change):
    cache, tables, q, *rest = step
    return (cache, tables, change(q.clone()), *rest)


# --------------------------------------------------------------------------------------------- slots of the weights
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths", [[(1, 90), (1, 30), (1, 50)], [(40, 90), (1, 30), (60, 50)], [(3, 90), (40, 30), (5, 50)]])
def test_slots_outside_the_weights_touch_nothing(ops, workspace, dtype, lengths):
    """A request whose slot is below 0 has no weights; one at or beyond their count is reported.  Neither touches their surroundings."""
    cache, tables, q, q_start, start_row, rows = make_step(1, lengths, 6, 2, 64, 16, dtype)
    pages, most = packed(ops, cache), max(rows)
    for slots, wrong in ((i32(-1, 1, 0), False), (i32(0, 3, -7), True), (i32(2 ** 31 - 1, 2, -2 ** 31), True)):
        around, out = torch.full((9, 2, most), 3.0, device=DEV), torch.empty(q.shape[0], 384, dtype=dtype, device=DEV)
        ops.packed_attention(q, out, pages, tables, q_start, start_row, max(n for n, _ in lengths), most, 6, 0.125, weights=around[3:6], seq_slot=slots,
                             add_weights=False, workspace=workspace)
        assert (ops.kernel_status() != 0) == wrong
        named = {int(s): i for i, s in enumerate(slots.tolist()) if 0 <= s < 3}
        for row in range(9):
            held = rows[named[row - 3]] if row - 3 in named else 0
            assert (around[row, :, held:] == 3).all() and (held == 0 or not (around[row, :, :held] == 3).any())
        assert out.float().isfinite().all()


def test_eviction_by_slots_outside_the_weights_keeps_nothing(ops, workspace):
    cache = ops.PackedPages.empty(12, 2, 16, 64, DEV)
    for t in (cache.k_codes, cache.v_codes):
        t.random_(0, 256)
    before = [t.clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    tables, to = torch.arange(8, dtype=torch.int32, device=DEV).view(4, 2), i32(8, 9, 10, 11)[:, None].contiguous()
    around, kept_around = torch.rand(9, 2, 30, device=DEV), torch.full((9, 2, 8), 5.0, device=DEV)
    kept = torch.full((4, 2, 8), 77, dtype=torch.int32, device=DEV)
    ops.packed_cache_evict(cache, tables, i32(30, 30, 6, 30), around[3:6], cache, to, kept, 8, seq_slot=i32(-1, 3, 1, 2 ** 31 - 1), kept_weights=kept_around[3:6],
                           workspace=workspace)
    assert ops.kernel_status() != 0
    assert (kept[[0, 1, 3]] == -1).all() and kept[2].tolist() == [[0, 1, 2, 3, 4, 5, -1, -1]] * 2
    assert torch.equal(kept_around[4, :, :6], around[4, :, :6])
    kept_around[4, :, :6] = 5.0
    assert (kept_around == 5).all()
    for a, b in zip(before, (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)):
        assert torch.equal(a[8:10], b[8:10]) and torch.equal(a[11], b[11])


def test_kept_weights_share_no_memory_with_the_weights(ops, workspace):
    from ferrisinfer_b200.errors import KernelError

    cache = ops.PackedPages.empty(8, 2, 16, 64, DEV)
    memory = torch.rand(2, 2, 2, 40, device=DEV)
    kept_rows = torch.zeros(2, 2, 8, dtype=torch.int32, device=DEV)
    call = lambda w, kept: ops.packed_cache_evict(cache, i32(0, 1, 2, 3).view(2, 2), i32(30, 20), w, cache, i32(4, 5).view(2, 1), kept_rows, 8,
                                                  kept_weights=kept, workspace=workspace)
    flat = memory.view(-1)
    for w, kept in ((memory[:, :, 0], memory[:, :, 0]), (memory[:, :, 0], memory[:, :, 0, 5:]), (memory[:, :, 0, 5:], memory[:, :, 0]),
                    (memory[:, :, 0], memory.flatten(2)[:, :, 39:50]), (flat[:160].view(2, 2, 40), flat[159:159 + 160].view(2, 2, 40)),
                    (flat[100:260].view(2, 2, 40), flat[:124].as_strided((2, 2, 8), (100, 10, 1)))):
        with pytest.raises(KernelError):
            call(w, kept)
    # rows between one another's, and one behind the other
    for w, kept in ((memory[:, :, 0], memory[:, :, 1]), (memory[:, :, 1], memory[:, :, 0]), (flat[:160].view(2, 2, 40), flat[160:].view(2, 2, 40)),
                    (memory[:, :, 0, 8:], memory[:, :, 0, :8])):
        old = w.clone()
        call(w, kept)
        assert torch.equal(w, old) and all(torch.equal(kept[s, h, :8], old[s, h][kept_rows[s, h].long()]) for s in range(2) for h in range(2))


# --------------------------------------------------------------------------------------------- scores of prompts
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths, empty", [([(150, 200)], (0, 128)), ([(40, 300), (150, 0)], (128, 256))])
def test_small_queries_and_a_block_of_rows_without_keys(ops, workspace, dtype, D, lengths, empty):
    """A block of 128 rows that has no page, or whose keys are all nought, beside queries of 1e-4 and less: numbers all the same."""
    step = make_step(3, lengths, 6, 2, D, 16, dtype)
    for small in (1e-4, 1e-20, 0.0):
        less = with_queries(step, lambda q: q * small)
        cache, tables = [t.clone() for t in less[0]], less[1].clone()
        pages = tables[0, empty[0] // 16:empty[1] // 16].long()
        for t in cache[:2]:
            t[pages] = 0  # scale, least and codes of the keys
        attend_and_compare(ops, workspace, (cache, *less[1:]), lengths, 6, 2, D, 16)
        tables[0, empty[0] // 16:empty[1] // 16] = -1
        attend_and_compare(ops, workspace, (less[0], tables, *less[2:]), lengths, 6, 2, D, 16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [0.0, -0.3])
@pytest.mark.parametrize("lengths", [[(150, 200), (1, 90)], [(1, 40), (1, 300)]])
def test_a_scale_that_is_nought_or_negative(ops, workspace, dtype, scale, lengths):
    for D in (64, 128):
        attend_and_compare(ops, workspace, make_step(4, lengths, 6, 2, D, 16, dtype), lengths, 6, 2, D, 16, scale=scale)


def test_a_scale_that_is_no_number_is_refused(ops, workspace):
    from ferrisinfer_b200.errors import KernelError

    for scale in (math.nan, math.inf, 3e38):
        with pytest.raises(KernelError):
            attend_and_compare(ops, workspace, make_step(4, [(1, 40)], 6, 2, 64, 16, torch.bfloat16), [(1, 40)], 6, 2, 64, 16, scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lengths", [[(300, 3000)], [(40, 0)], [(90, 700), (1, 2000)]])
def test_queries_that_are_not_numbers(ops, workspace, dtype, D, lengths):
    """NaN in a query is NaN in its output, however many blocks share the row's cached rows."""
    def spoil(q):
        q[5, 3], q[17, 4 * D + 1] = math.nan, math.nan
        return q

    attend_and_compare(ops, workspace, with_queries(make_step(5, lengths, 6, 2, D, 16, dtype), spoil), lengths, 6, 2, D, 16)


# --------------------------------------------------------------------------------------------- bounds that are not tight
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, kv_heads, D, n", [(28, 4, 128, 1), (14, 2, 64, 1), (6, 2, 64, 2), (12, 1, 128, 1), (24, 1, 64, 1)])
@pytest.mark.parametrize("max_q", [17, 512])
def test_a_most_of_queries_that_no_request_reaches(ops, workspace, dtype, heads, kv_heads, D, n, max_q):
    for lengths in ([(n, 90)], [(n, 90), (1, 300)]):
        attend_and_compare(ops, workspace, make_step(7, lengths, heads, kv_heads, D, 16, dtype), lengths, heads, kv_heads, D, 16, max_q=max_q)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("max_q", [2 ** 30, 2 ** 40])
def test_a_most_of_queries_beyond_32_bits(ops, workspace, dtype, max_q):
    for lengths in ([(1, 90)], [(70, 90), (1, 300)]):
        attend_and_compare(ops, workspace, make_step(7, lengths, 6, 2, 64, 16, dtype), lengths, 6, 2, 64, 16, max_q=max_q)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths", [[(1, 90), (1, 300)], [(70, 30), (1, 300)]])
def test_a_most_of_rows_that_no_request_reaches(ops, workspace, dtype, lengths):
    for max_kv in (10 ** 6, 2 ** 31 - 1, 2 ** 40):
        attend_and_compare(ops, workspace, make_step(8, lengths, 6, 2, 64, 16, dtype), lengths, 6, 2, 64, 16, max_kv=max_kv)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [1, 40])
def test_no_rows_at_all(ops, workspace, dtype, n):
    """A caller who says that no request has a row: outputs of nought, no weight touched."""
    cache, tables, q, q_start, start_row, rows = make_step(9, [(n, 20)], 4, 2, 64, 16, dtype)
    out, weights = torch.full((n, 256), 7.0, dtype=dtype, device=DEV), torch.full((1, 2, 30), 3.0, device=DEV)
    ops.packed_attention(q, out, packed(ops, cache), tables, q_start, start_row, n, 0, 4, 0.125, weights=weights, workspace=workspace)
    assert (out == 0).all() and (weights == 3).all()


def test_numbers_that_the_library_cannot_take(ops, workspace):
    from ferrisinfer_b200.errors import KernelError

    lengths = [(1, 90), (1, 300)]
    step = make_step(8, lengths, 6, 2, 64, 16, torch.bfloat16)
    attend_and_compare(ops, workspace, step, lengths, 6, 2, 64, 16, window=2 ** 40)  # (a window that holds everything)
    with pytest.raises(KernelError):
        attend_and_compare(ops, workspace, step, lengths, 6, 2, 64, 16, scale=1e300)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, others", [(6, [(1, 50)]), (6, [(40, 50)]), (6, [(40, 50), (1, 20)]), (40, [(40, 50)]), (40, [(1, 50)])])
@pytest.mark.parametrize("add", [True, False])
def test_a_request_without_queries_keeps_its_weights(ops, workspace, dtype, heads, others, add):
    lengths = [(0, 100), *others]
    cache, tables, q, q_start, start_row, rows = make_step(10, lengths, heads, 2, 64, 16, dtype)
    out, weights = torch.empty(q.shape[0], heads * 64, dtype=dtype, device=DEV), torch.full((len(lengths), 2, max(rows)), 3.0, device=DEV)
    ops.packed_attention(q, out, packed(ops, cache), tables, q_start, start_row, max(n for n, _ in lengths), max(rows), heads, 0.125,
                         weights=weights, add_weights=add, workspace=workspace)
    assert (weights[0] == 3).all() and (weights[1, :, :50] != 3).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("queries", [1, 40])
def test_many_small_weights_beside_a_great_one(ops, workspace, D, queries):
    """2,000 rows of weight e^-15 and one that takes the rest with a value of nought: what the many say is all there is."""
    n, gap = 2000, 15.0
    k, v = torch.zeros(n + queries, 1, D, device=DEV), torch.ones(n + queries, 1, D, device=DEV)
    k[0], v[0] = 1.0, 0.0
    cache, table = plain.cache_of(k, v, 16), torch.arange(-(-(n + queries) // 16), dtype=torch.int32, device=DEV)[None].contiguous()
    q = torch.full((queries, 6 * D), gap / 4, dtype=torch.bfloat16, device=DEV)
    scale = 4.0 / D  # the first row's score is `gap`, the others' are nought
    step = (cache, table, q, i32(0, queries), i32(n), [n + queries])
    attend_and_compare(ops, workspace, step, [(queries, n)], 6, 1, D, 16, scale=scale)


# --------------------------------------------------------------------------------------------- values of all sizes
@pytest.mark.parametrize("heads, kv_heads, D", [(4, 2, 64), (6, 1, 128), (12, 1, 64), (2, 1, 96), (2, 1, 256)])
@pytest.mark.parametrize("small", [2.0 ** -8, 2.0 ** -16, 2.0 ** -40])
def test_32_bit_rows_keep_their_bits_beside_greater_values(ops, workspace, heads, kv_heads, D, small):
    """The second group of a head is `small` times the first, and one row is as many times greater than all others in every group, with
    a key that no query looks for: its share is nothing."""
    lengths = [(1, 700), (3, 90), (1, 40)]
    cache, tables, *rest = make_step(6, lengths, heads, kv_heads, D, 16, torch.float32)
    cache[3][..., 1, :] *= small
    scale = 0.05 * D ** -0.5
    attend_and_compare(ops, workspace, (cache, tables, *rest), lengths, heads, kv_heads, D, 16, scale=scale)
    page = int(tables[0, 1])
    cache[3][page, :, 7] /= small
    rest[0].abs_()
    cache[1][page, :, 7] = torch.tensor([0.0, -400.0], device=DEV)  # (scale, least): a score more than a hundred below the others'
    attend_and_compare(ops, workspace, (cache, tables, *rest), lengths, heads, kv_heads, D, 16, scale=scale, far=[(0, 23)])


# --------------------------------------------------------------------------------------------- eviction
def kept_of(weights, there, budget, keep_first, keep_last):
    """``plain.kept`` where row r stands only if there[r]."""
    n = len(weights)
    rows = [r for r in range(n) if there[r]]
    if len(rows) <= budget:
        return rows

    def rank(r):
        if r < keep_first or r >= n - keep_last:
            return (0, 0.0, r)
        w = weights[r]
        return (1, 0.0, r) if math.isnan(w) else (2, -w, r)

    return sorted(sorted(rows, key=rank)[:budget])


@pytest.mark.parametrize("rows, budget, first, last, page_size, width", [
    ([60, 90], 64, 4, 8, 16, 6),        # all that is there stays, or what is there is no more than the budget
    ([500, 300, 0], 64, 20, 40, 16, 32),
    ([1500, 260], 1400, 4, 8, 7, 215),  # fewer rows there than the budget, more rows than it
    ([20000], 700, 100, 300, 16, 1250),  # several blocks to a request
    ([20000], 19000, 0, 0, 64, 313),
    ([200, 100], 32, 4, 8, 16, 8),      # a table that ends before the rows do
])
@pytest.mark.parametrize("kind", ["spread", "ties", "special"])
def test_rows_without_a_page_are_not_there_to_be_kept(ops, workspace, rows, budget, first, last, page_size, width, kind):
    gen = torch.Generator(device=DEV).manual_seed(budget + len(kind))
    S, most, hkv, D = len(rows), max(rows), 2, 64
    to_blocks = -(-budget // page_size)
    pages = S * (width + to_blocks)
    cache = ops.PackedPages.empty(pages, hkv, page_size, D, DEV)
    for name in ("k_codes", "v_codes"):
        getattr(cache, name).random_(0, 256, generator=gen)
    for name in ("k_scales", "v_scales"):
        t = getattr(cache, name)
        t.copy_(torch.randn(t.shape, generator=gen, device=DEV).abs())
    ids = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    tables, to_tables = ids[:S * width].view(S, width).clone(), ids[S * width:].view(S, to_blocks).contiguous()
    tables[torch.rand(S, width, generator=gen, device=DEV) < 0.3] = -1
    tables[0, 0], tables[0, 1] = -1, int(ids[1])
    w = torch.rand(S, hkv, most, generator=gen, device=DEV)
    if kind == "ties":
        w = (w * 4).floor()
    elif kind == "special":
        w[w < 0.05] = math.nan
        w[(w > 0.05) & (w < 0.1)] = math.inf
        w[(w > 0.1) & (w < 0.2)] = -math.inf
    kept_rows, kept_w = torch.full((S, hkv, budget), 77, dtype=torch.int32, device=DEV), torch.full((S, hkv, budget + 2), 5.0, device=DEV)
    tensors = (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)
    old = [t.clone() for t in tensors]
    ops.packed_cache_evict(cache, tables, i32(*rows), w, cache, to_tables, kept_rows, budget, keep_first=first, keep_last=last, kept_weights=kept_w,
                           workspace=workspace)
    for s, n in enumerate(rows):
        table = tables[s].tolist() + [-1] * (n // page_size + 1)
        there = [table[r // page_size] >= 0 for r in range(n)]
        for h in range(hkv):
            want = kept_of(w[s, h, :n].tolist(), there, budget, first, last)
            assert kept_rows[s, h].tolist() == want + [-1] * (budget - len(want))
            src, at = torch.tensor(want, dtype=torch.long, device=DEV), torch.arange(len(want), device=DEV)
            assert torch.equal(kept_w[s, h, :len(want)].nan_to_num(-3), w[s, h][src].nan_to_num(-3))
            assert (kept_w[s, h, len(want):] == 5).all()
            for a, b in zip(old, tensors):
                assert torch.equal(a[tables[s].long()[src // page_size], h, src % page_size], b[to_tables[s].long()[at // page_size], h, at % page_size])
    for a, b in zip(old, tensors):  # what was read stays as it was
        live = tables[tables >= 0].long()
        assert torch.equal(a[live], b[live])


def test_eviction_says_when_weights_end_before_the_rows(ops, workspace):
    cache = ops.PackedPages.empty(8, 1, 16, 64, DEV)
    kept_rows = torch.empty(1, 1, 10, dtype=torch.int32, device=DEV)
    ops.packed_cache_evict(cache, i32(0, 1, 2, 3)[None].contiguous(), i32(60), torch.rand(1, 1, 50, device=DEV), cache, i32(4)[None].contiguous(),
                           kept_rows, 10, workspace=workspace)
    assert ops.kernel_status() != 0


# --------------------------------------------------------------------------------------------- many requests, long ones
@pytest.mark.parametrize("D", [64, 128])
def test_more_requests_than_are_dealt_out_evenly_and_a_prompt(ops, workspace, D):
    lengths = [(1, i % 3) for i in range(1100)] + [(70, 30)] + [(1, 5)] * 3
    attend_and_compare(ops, workspace, make_step(11, lengths, 4, 2, D, 16, torch.bfloat16), lengths, 4, 2, D, 16)


def test_more_pairs_of_tiles_than_are_dealt_out_evenly(ops, workspace):
    lengths = [(3, i % 4) for i in range(1030)]  # 18 query rows of a kv head each, a pair of tiles of their own
    attend_and_compare(ops, workspace, make_step(12, lengths, 6, 1, 64, 16, torch.bfloat16), lengths, 6, 1, 64, 16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_more_scores_than_are_kept(ops, workspace, dtype):
    """Tables so wide that the scores of a step would fill more than 512 MB: the weights come from scores formed again."""
    lengths = [(1, 100 + i) for i in range(40)]
    cache, tables, *rest = make_step(13, lengths, 8, 4, 64, 16, dtype)
    wide = torch.full((len(lengths), 8192), -1, dtype=torch.int32, device=DEV)
    wide[:, :tables.shape[1]] = tables
    q, q_start, start_row, rows = rest
    out, weights = torch.empty(40, 512, dtype=dtype, device=DEV), torch.zeros(40, 4, 131072, device=DEV)
    ops.packed_attention(q, out, packed(ops, cache), wide, q_start, start_row, 1, 131072, 8, 0.125, weights=weights, workspace=workspace)
    other, same = torch.empty_like(out), torch.zeros(40, 4, max(rows), device=DEV)
    ops.packed_attention(q, other, packed(ops, cache), tables, q_start, start_row, 1, max(rows), 8, 0.125, weights=same, workspace=workspace)
    # The same scores and sums, cut into other pieces: 24-bit sums of a few hundred weights, then the type's rounding.
    assert (out.double() - other.double()).abs().max() <= other.double().abs().max() * (2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -18)
    assert ((weights[:, :, :max(rows)] - same).abs() <= same * 2.0 ** -18).all() and (weights[:, :, max(rows):] == 0).all()


@pytest.mark.parametrize("D", [64, 128])
def test_long_runs_of_prompts_are_cut_and_joined(ops, workspace, D):
    """Portions after so many rows that a CTA goes on from one pair of tiles to the next, against a call for each alone."""
    lengths = [(130, 40000), (200, 30000), (64, 65000), (3, 9000)]
    gen = torch.Generator(device=DEV).manual_seed(14)
    rows, ps = [n + s for n, s in lengths], 64
    blocks = [-(-r // ps) for r in rows]
    cache = []
    for _ in range(2):
        cache.append(torch.randint(0, 256, (sum(blocks), 1, ps, D // 2), generator=gen, device=DEV, dtype=torch.uint8))
        scale = 0.05 + 0.2 * torch.rand(sum(blocks), 1, ps, D // 32, generator=gen, device=DEV)
        cache.append(torch.stack([scale, -7.5 * scale], -1).to(torch.bfloat16))
    ids = torch.randperm(sum(blocks), generator=gen, device=DEV).to(torch.int32)
    tables = torch.full((len(lengths), max(blocks)), -1, dtype=torch.int32, device=DEV)
    starts = [0]
    for i, b in enumerate(blocks):
        tables[i, :b] = ids[sum(blocks[:i]):sum(blocks[:i + 1])]
        starts.append(starts[-1] + lengths[i][0])
    q = torch.randn(starts[-1], 7 * D, generator=gen, device=DEV).bfloat16()
    out, weights = torch.empty_like(q), torch.zeros(len(lengths), 1, max(rows), device=DEV)
    pages = packed(ops, cache)
    ops.packed_attention(q, out, pages, tables, i32(*starts), i32(*(s for _, s in lengths)), 200, max(rows), 7, D ** -0.5, weights=weights,
                         workspace=workspace)
    for i, (n, start) in enumerate(lengths):
        k, v, _ = plain.request_rows(cache, tables[i], rows[i], ps)
        mine = q[starts[i]:starts[i + 1]].double().view(n, 7, D).transpose(0, 1)
        s = (mine @ k[:, 0].t()) * D ** -0.5
        s.masked_fill_(torch.arange(rows[i], device=DEV) > start + torch.arange(n, device=DEV)[:, None], -math.inf)
        p = torch.softmax(s, -1)
        want, got = (p @ v[:, 0]).transpose(0, 1), out[starts[i]:starts[i + 1]].double().view(n, 7, D)
        # bf16 rows: the result's rounding (2^-9 on average) and weights and values in eleven bits
        assert (got - want).norm() <= 2.0 ** -8 * want.norm()
        w = p.sum((0, 1))
        assert ((weights[i, 0, :rows[i]].double() - w).abs() <= w * 2.0 ** -14).all()


@pytest.mark.parametrize("heads, kv_heads, D, n", [(4, 2, 64, 3), (6, 1, 128, 1), (12, 1, 64, 1), (2, 1, 96, 4), (2, 1, 256, 8)])
@pytest.mark.parametrize("small", [2.0 ** -8, 2.0 ** -24, 2.0 ** -40])
def test_few_bf16_rows_keep_small_groups_beside_great_ones(ops, workspace, heads, kv_heads, D, n, small):
    """The second group of a head is `small` times the others, in steps that the kernel for few rows takes."""
    lengths = [(1, 700), (n, 90), (1, 40)]
    cache, tables, *rest = make_step(15, lengths, heads, kv_heads, D, 16, torch.bfloat16)
    cache[3][..., 1, :] *= small
    attend_and_compare(ops, workspace, (cache, tables, *rest), lengths, heads, kv_heads, D, 16, scale=0.05 * D ** -0.5)
