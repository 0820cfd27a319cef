"""The paged cache in 4 bits against its plain form in 64 bits: writing, reading, attention with the rows' weights, eviction."""

import math

import pytest
import torch

import plain_packed as plain

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


def rng(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def packed(ops, tensors):
    return ops.PackedPages(*(t.to(DEV) for t in tensors))


# --------------------------------------------------------------------------------------------- write, read
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens, kv_heads, D, page_size, offset", [
    (1, 1, 32, 16, 0), (3, 2, 64, 16, 0), (37, 3, 96, 24, 0), (65, 2, 128, 7, 0), (17, 1, 256, 64, 0),
    (5, 2, 64, 16, 1), (9, 4, 128, 16, 3), (33, 1, 160, 1, 0),  # (columns off 16 bytes; pages of one row)
])
def test_write_and_read(ops, dtype, tokens, kv_heads, D, page_size, offset):
    gen = rng(tokens + D)
    width = kv_heads * D
    both = torch.randn(tokens, 2 * width + offset, generator=gen, device=DEV) * 3 + torch.randn(1, 2 * width + offset, generator=gen, device=DEV) * 20
    both[:, ::7] *= 1e-3
    both = both.to(dtype)
    k, v = both[:, offset:offset + width], both[:, offset + width:]
    pages = -(-tokens // page_size) + 2
    cache = ops.PackedPages.empty(pages, kv_heads, page_size, D, DEV)
    for t in (cache.k_codes, cache.v_codes):
        t.fill_(0x5A)
    slots = torch.randperm(pages * page_size, generator=gen, device=DEV)[:tokens].to(torch.int32)
    if tokens > 2:
        slots[1] = -1
    ops.packed_cache_write(k, v, slots, cache)
    at = slots.long().clamp(min=0)
    live = slots >= 0
    for x, codes, scales, keys in ((k, cache.k_codes, cache.k_scales, True), (v, cache.v_codes, cache.v_scales, False)):
        rows = x.reshape(tokens, kv_heads, D)
        got_codes = plain.codes_of(codes[at // page_size, :, at % page_size], keys)[live]
        got_scales = scales[at // page_size, :, at % page_size][live]
        want = plain.scales_of(rows)[live]
        assert torch.equal(got_scales, want)
        s = want.double()
        exact = (rows.double()[live] - s[..., 1].repeat_interleave(32, -1)) / s[..., 0].repeat_interleave(32, -1)
        # the kernel's x - least and its quotient are rounded to 24 bits: within 2^-22 of a tie either side is right
        assert ((got_codes - exact.clamp(0, 15)).abs() <= 0.5 + 2.0 ** -18).all()
    # every row that was not named keeps what it held
    untouched = torch.ones(pages * page_size, dtype=torch.bool, device=DEV)
    untouched[at[live]] = False
    rows = untouched.nonzero()[:, 0]
    assert (cache.k_codes[rows // page_size, :, rows % page_size] == 0x5A).all()
    assert (cache.v_scales[rows // page_size, :, rows % page_size] == 0).all()
    # reading gives what the rows stand for, rounded once, and zeros for no row
    back = torch.full((tokens, 2 * width + offset), 9.0, device=DEV, dtype=dtype)
    ops.packed_cache_read(cache, slots, back[:, offset:offset + width], back[:, offset + width:])
    for name, x, keys in (("k", back[:, offset:offset + width], True), ("v", back[:, offset + width:], False)):
        stands = plain.values(getattr(cache, name + "_codes")[at // page_size, :, at % page_size],
                              getattr(cache, name + "_scales")[at // page_size, :, at % page_size], keys)
        stands = torch.where(live[:, None, None], stands, 0.0).flatten(1)
        # scale * code is exact in 32 bits, its sum with the least is rounded, then once more to the type: bit for bit
        assert torch.equal(x, stands.float().to(dtype))
    if offset:
        assert (back[:, :offset] == 9).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_groups_of_special_values(ops, dtype):
    x = torch.randn(10, 64, generator=rng(3), device=DEV)
    x[0] = 0.0
    x[1] = 100.0
    x[2, :32] = 100.0 + torch.arange(32, device=DEV) * 0.5
    x[3, 5] = math.nan
    x[4, 40] = math.inf
    x[5, 40] = -math.inf
    x[6] = 1e38
    x[6, 3] = -3e38
    x[7] *= 1e-38
    x[8] = -7.0
    x[9] = 3e38
    x = x.to(dtype)
    cache = ops.PackedPages.empty(1, 1, 16, 64, DEV)
    slots = torch.arange(10, dtype=torch.int32, device=DEV)
    ops.packed_cache_write(x, x, slots, cache)
    back = torch.empty(10, 64, device=DEV)
    also = torch.empty_like(back)
    ops.packed_cache_read(cache, slots, back, also)
    assert torch.equal(torch.nan_to_num(back, 1.5), torch.nan_to_num(also, 1.5))
    want = torch.zeros(10, 64, dtype=torch.bool, device=DEV)
    want[3, :32] = want[4, 32:] = want[5, 32:] = True  # the whole group stands as NaN, the other one does not
    want[6, :32] = torch.isinf(torch.tensor(1e38).to(dtype).float() + 3e38).item()  # a spread of no 32-bit number
    assert torch.equal(torch.isnan(back), want)
    for r in (0, 8):
        assert torch.equal(back[r], x[r].float())
    assert (back[1] - 100).abs().max() == 0 and (back[9] / x[9].float() - 1).abs().max() < 2.0 ** -7
    # an offset far larger than the spread: half a step of the spread above the rounded least
    assert (back[2, :32] - x[2, :32].float()).abs().max() <= 0.5 * (15.5 + 0.5) / 15 * (1 + 2.0 ** -8)


# --------------------------------------------------------------------------------------------- attention
def make_step(seed, lengths, heads, kv_heads, D, page_size, dtype, offset=0, holes=()):
    """A step of requests (queries, rows before them): packed cache, tables (pages in no order, unused rows NaN), queries."""
    gen = rng(seed)
    rows = [max(q + s, 0) for q, s in lengths]  # what the request holds after the step
    blocks = [max(1, -(-r // page_size)) for r in rows]
    order = torch.randperm(sum(blocks) + 1, generator=gen, device=DEV).tolist()
    tables = torch.full((len(lengths), max(blocks) + 1), -1, dtype=torch.int32, device=DEV)
    at, parts = 0, None
    for i, (r, b) in enumerate(zip(rows, blocks)):
        mine = order[at:at + b]
        at += b
        k = torch.randn(b * page_size, kv_heads, D, generator=gen, device=DEV) + torch.randn(kv_heads, D, generator=gen, device=DEV)
        v = torch.randn(b * page_size, kv_heads, D, generator=gen, device=DEV)
        one = plain.cache_of(k[:r], v[:r], page_size, pages=sum(blocks) + 1, order=mine) if r else None
        if one is not None:
            if parts is None:
                parts = one
            else:
                for a, o in zip(parts, one):
                    a[mine] = o[mine]
        tables[i, :b] = torch.tensor(mine, dtype=torch.int32)
    for i, b in holes:
        tables[i, b] = -1
    T = sum(q for q, _ in lengths)
    q = torch.randn(T, heads * D + offset, generator=gen, device=DEV).to(dtype)[:, offset:]
    starts = [0]
    for n, _ in lengths:
        starts.append(starts[-1] + n)
    return parts, tables, q, torch.tensor(starts, dtype=torch.int32, device=DEV), torch.tensor([s for _, s in lengths], dtype=torch.int32, device=DEV), rows


def check_step(ops, workspace, lengths, heads, kv_heads, D, page_size, dtype, window=0, seed=0, offset=0, holes=(), spoil=None, add=True,
               slots=False, scale=None):
    cache, tables, q, q_start, start_row, rows = make_step(seed, lengths, heads, kv_heads, D, page_size, dtype, offset, holes)
    if spoil is not None:
        spoil(cache, tables)
    scale = D ** -0.5 if scale is None else scale
    pages = packed(ops, cache)
    T, S = q.shape[0], len(lengths)
    out = torch.full((T, heads * D + offset), 7.0, dtype=dtype, device=DEV)[:, offset:]
    most = max(rows)
    gen = rng(seed + 1)
    weights = torch.rand(S + 2, kv_heads, most + 3, generator=gen, device=DEV)
    before = weights.clone()
    slot = torch.randperm(S + 2, generator=gen, device=DEV)[:S].to(torch.int32) if slots else None
    ops.packed_attention(q, out, pages, tables, q_start, start_row, max(n for n, _ in lengths), most, heads, scale, window=window,
                         weights=weights, seq_slot=slot, add_weights=add, workspace=workspace)
    alone = torch.full_like(out, 7.0)
    ops.packed_attention(q, alone, pages, tables, q_start, start_row, max(n for n, _ in lengths), most, heads, scale, window=window,
                         workspace=workspace)
    at = 0
    kept = torch.zeros_like(weights, dtype=torch.bool)
    for i, ((n, start), r) in enumerate(zip(lengths, rows)):
        k, v, has = plain.request_rows(cache, tables[i], r, page_size)
        want, w, size, spread = plain.attend(q[at:at + n].double().view(n, heads, D), k, v, has, start, scale, window)
        # Scores: a sum of D / 8 + 8 steps of 24-bit numbers (the tensor cores cut rather than round: a whole unit each).  Twice,
        # in a weight and in the sum that it is divided by, and the exponential and sums of the weights beside them.
        rel = (D / 8 + 8) * 2.0 ** -23 * spread * 2 + 2.0 ** -19
        # Outputs: weights, and their products with scales, rounded to eight bits for bf16 rows (off by at most 2^-8 of each
        # and to both sides: half of that for their sum), then the result once more.
        lossy = 2.0 ** -9 if dtype == torch.bfloat16 else 0.0
        least = torch.zeros(n, heads, 1, dtype=torch.float64, device=DEV)
        if n and r:
            s = cache[3].double().nan_to_num(0.0)
            least = least + (s[..., 1].abs() * 2).max()
        bound = (size + least) * (rel[..., None] + lossy) + want.abs() * (lossy + 2.0 ** -23) + 1e-30
        for got in (out, alone):
            g = got[at:at + n].double().view(n, heads, D)
            nan = torch.isnan(want)
            assert torch.equal(torch.isnan(g), nan), (i, (torch.isnan(g) != nan).nonzero()[:4])
            assert ((g - want).abs() <= bound)[~nan].all(), (i, ((g - want).abs() / bound)[~nan].max())
        row = i if slot is None else int(slot[i])
        held = max(start, 0)
        base = before[row, :, :r].double().clone()
        base[:, held:] = 0
        total = w + (base if add else 0)
        e = rel.nan_to_num(0.0).max() if rel.numel() else torch.zeros((), device=DEV)  # (of the queries that see numbers)
        g = weights[row, :, :r].double()
        nan = torch.isnan(total)
        assert torch.equal(torch.isnan(g), nan)
        assert ((g - total).abs() <= w * e + total * 2.0 ** -20 + 1e-30)[~nan].all(), (i, ((g - total).abs() - w * e).nan_to_num().max())
        kept[row, :, :r] = True
        at += n
    assert torch.equal(weights[~kept], before[~kept])  # nothing beyond the requests' rows


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, kv_heads, D, page_size", [
    (1, 1, 32, 16), (14, 2, 64, 16), (6, 3, 96, 24), (12, 2, 128, 16), (28, 4, 128, 64), (4, 2, 192, 7), (8, 1, 256, 16), (20, 1, 64, 32),
    (33, 3, 32, 1),
])
def test_single_tokens(ops, workspace, dtype, heads, kv_heads, D, page_size):
    check_step(ops, workspace, [(1, 0), (1, 1), (1, 15), (1, 16), (1, 63), (1, 300)], heads, kv_heads, D, page_size, dtype, seed=D)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths, window", [
    ([(5, 0), (1, 40), (0, 9), (33, 0), (2, 100)], 0),
    ([(17, 3), (1, 0), (40, 64)], 0),
    ([(17, 30), (1, 50), (40, 0)], 5),
    ([(3, 200), (1, 200)], 64),
    ([(1, 20), (1, 700), (1, 3)], 1),
    ([(130, 70)], 0),
    ([(257, 0), (64, 129)], 100),
])
@pytest.mark.parametrize("heads, kv_heads, D, page_size", [(6, 2, 64, 16), (7, 1, 128, 24)])
def test_portions(ops, workspace, dtype, lengths, window, heads, kv_heads, D, page_size):
    check_step(ops, workspace, lengths, heads, kv_heads, D, page_size, dtype, window=window, seed=len(lengths), offset=8, slots=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, kv_heads, D", [(14, 2, 64), (12, 2, 128)])
def test_long_requests_are_cut_and_joined(ops, workspace, dtype, heads, kv_heads, D):
    check_step(ops, workspace, [(1, 4099), (1, 0), (1, 2047)], heads, kv_heads, D, 16, dtype, seed=5, add=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_without_a_page_and_queries_that_see_nothing(ops, workspace, dtype):
    # a hole in the middle, a request without any page, requests that begin before their first row
    check_step(ops, workspace, [(1, 100), (1, 30), (3, 40), (1, -1), (4, -3)], 4, 2, 64, 16, dtype, seed=9,
               holes=[(0, 2), (0, 3), (1, 0), (1, 1), (2, 0)])
    check_step(ops, workspace, [(20, 100), (40, -17)], 4, 2, 128, 16, dtype, seed=10, holes=[(0, 0), (0, 1), (0, 2), (0, 3)], window=48)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("which", ["keys", "values"])
@pytest.mark.parametrize("lengths", [[(1, 70), (1, 40)], [(30, 20), (9, 0)], [(150, 10)]])
def test_rows_that_are_not_finite_reach_those_that_see_them_only(ops, workspace, dtype, which, lengths):
    def spoil(cache, tables):
        page = int(tables[0, 2])  # rows 32 .. 47 of the first request: two groups of one of them, and one behind all of them
        cache[1 if which == "keys" else 3][page, 1, 5, 1] = math.nan
        cache[1 if which == "keys" else 3][page, 0, 9, 0, 0] = math.nan

    check_step(ops, workspace, lengths, 6, 2, 64, 16, dtype, seed=4, spoil=spoil)
    check_step(ops, workspace, lengths, 6, 2, 64, 16, dtype, seed=4, spoil=spoil, window=3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scores_far_apart_and_scales_of_all_sizes(ops, workspace, dtype):
    def spoil(cache, tables):  # keys of one request a thousand times as large, values of very different sizes
        cache[1][int(tables[0, 0])] *= 1000
        cache[3][int(tables[1, 0])] *= 1e-6
        cache[3][int(tables[1, 1])] *= 1e6

    check_step(ops, workspace, [(1, 40), (1, 40)], 4, 2, 64, 16, dtype, seed=6, spoil=spoil)
    check_step(ops, workspace, [(37, 40), (20, 40)], 4, 2, 64, 16, dtype, seed=6, spoil=spoil)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, kv_heads, D, queries", [(7, 1, 64, 1), (4, 1, 128, 1), (2, 1, 96, 3), (8, 1, 64, 9)])
def test_sums_over_very_many_rows(ops, workspace, dtype, heads, kv_heads, D, queries):
    """70,000 rows of nearly equal weight, so that the output is small beside what is added up."""
    gen, n, ps = rng(D), 70000, 16
    pages = -(-n // ps)
    cache = []
    for _ in range(2):
        cache.append(torch.randint(0, 256, (pages, kv_heads, ps, D // 2), generator=gen, device=DEV, dtype=torch.uint8))
        scale = 0.05 + 0.3 * torch.rand(pages, kv_heads, ps, D // 32, generator=gen, device=DEV)
        cache.append(torch.stack([scale, -7.5 * scale], -1).to(torch.bfloat16))
    tables = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)[None].contiguous()
    q = torch.randn(queries, heads * D, generator=gen, device=DEV).to(dtype)
    out, weights = torch.empty_like(q), torch.zeros(1, kv_heads, n, device=DEV)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    ops.packed_attention(q, out, packed(ops, cache), tables, i32(0, queries), i32(n - queries), queries, n, heads, 0.3 * D ** -0.5, weights=weights,
                         workspace=workspace)
    k, v, has = plain.request_rows(cache, tables[0], n, ps)
    want, w, _, _ = plain.attend(q.double().view(queries, heads, D), k, v, has, n - queries, 0.3 * D ** -0.5)
    off = (out.double().view(queries, heads, D) - want).norm() / want.norm()
    # 32-bit rows: scores and weights within a few 2^-23, sums of 16 to 32 rows cut off at 24 bits, those added up in rounded fp32 over
    # some thousand places in turn, errors of both signs; bf16 rows: the result's rounding (2^-9 on average, at most 2^-8 of each number)
    # and weights in eleven bits.
    assert off < (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -18), off
    assert ((weights[0].double() - w).abs() / w).max() < 2.0 ** -15 and (weights[0].double() - w).norm() / w.norm() < 2.0 ** -18


def test_same_bits_from_run_to_run(ops, workspace):
    cache, tables, q, q_start, start_row, rows = make_step(2, [(1, 900), (1, 2500)], 12, 2, 128, 16, torch.bfloat16)
    pages, seen = packed(ops, cache), []
    for _ in range(3):
        out, weights = torch.empty_like(q), torch.zeros(2, 2, max(rows), device=DEV)
        ops.packed_attention(q, out, pages, tables, q_start, start_row, 1, max(rows), 12, 128 ** -0.5, weights=weights, workspace=workspace)
        seen.append((out, weights))
    assert all(torch.equal(a, b) for one in seen[1:] for a, b in zip(seen[0], one))


@pytest.mark.parametrize("lengths", [[(1, 500), (1, 90)], [(70, 300), (1, 100), (3, 9)]])
def test_rows_beyond_what_the_caller_names_are_not_seen(ops, workspace, lengths):
    cache, tables, q, q_start, start_row, rows = make_step(3, lengths, 6, 2, 64, 16, torch.bfloat16)
    most, at = 200, 0
    out, weights = torch.empty_like(q), torch.zeros(len(lengths), 2, most, device=DEV)
    ops.packed_attention(q, out, packed(ops, cache), tables, q_start, start_row, max(n for n, _ in lengths), most, 6, 0.125, weights=weights, workspace=workspace)
    for i, ((n, start), r) in enumerate(zip(lengths, rows)):
        k, v, has = plain.request_rows(cache, tables[i], r, 16)
        has[most:] = False
        want, w, size, _ = plain.attend(q[at:at + n].double().view(n, 6, 64), k, v, has, start, 0.125)
        got = out[at:at + n].double().view(n, 6, 64)
        assert ((got - want).abs() <= (size + 4) * 2.0 ** -10 + want.abs() * 2.0 ** -8).all()
        held = min(r, most)
        assert ((weights[i, :, :held].double() - w[:, :held]).abs() <= w[:, :held] * 2.0 ** -14 + 1e-12).all()
        at += n


def test_on_another_stream(ops, workspace):
    check_step(ops, workspace, [(1, 90)], 4, 2, 64, 16, torch.bfloat16)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        check_step(ops, workspace, [(1, 90), (5, 30)], 4, 2, 64, 16, torch.bfloat16)
    torch.cuda.current_stream().wait_stream(stream)


# --------------------------------------------------------------------------------------------- eviction
@pytest.mark.parametrize("rows, budget, first, last, kv_heads, D, page_size, to_size", [
    ([40], 16, 0, 0, 1, 32, 16, 16),
    ([1, 0, 33, 64, 65, 200], 64, 4, 16, 2, 64, 16, 16),
    ([1500, 999, 31], 257, 1, 100, 3, 96, 24, 16),
    ([5000], 4096, 4, 1024, 2, 128, 16, 64),
    ([70, 80], 1, 0, 1, 1, 64, 16, 7),
    ([70, 80], 1, 1, 0, 1, 64, 7, 16),
    ([1025, 2049], 30, 30, 0, 2, 256, 16, 16),
    ([9000, 20000], 700, 0, 0, 1, 64, 16, 16),
])
@pytest.mark.parametrize("kind", ["spread", "ties", "nought", "special"])
def test_eviction(ops, workspace, rows, budget, first, last, kv_heads, D, page_size, to_size, kind):
    gen = rng(budget + len(kind))
    S, most = len(rows), max(rows)
    blocks, to_blocks = -(-most // page_size), -(-budget // to_size)
    same = page_size == to_size
    pages = S * blocks + (S * to_blocks if same else 0)
    cache = ops.PackedPages.empty(pages, kv_heads, page_size, D, DEV)
    for name in ("k_codes", "v_codes"):
        getattr(cache, name).random_(0, 256, generator=gen)
    for name in ("k_scales", "v_scales"):
        t = getattr(cache, name)
        t.copy_(torch.randn(t.shape, generator=gen, device=DEV))
    to = cache if same else ops.PackedPages.empty(S * to_blocks, kv_heads, to_size, D, DEV)
    ids = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    tables = ids[:S * blocks].view(S, blocks).contiguous()
    to_tables = (ids[S * blocks:] if same else torch.randperm(S * to_blocks, generator=gen, device=DEV).to(torch.int32)).view(S, to_blocks).contiguous()
    w = torch.rand(S + 1, kv_heads, most + 5, generator=gen, device=DEV)
    if kind == "ties":
        w = (w * 4).floor()
    elif kind == "nought":
        w = torch.where(w < 0.98, 0.0, w) * torch.where(w < 0.5, -1.0, 1.0)  # -0 among the noughts
    elif kind == "special":
        w[w < 0.05] = math.nan
        w[(w > 0.05) & (w < 0.1)] = math.inf
        w[(w > 0.1) & (w < 0.2)] = -math.inf
        w[(w > 0.2) & (w < 0.3)] *= 1e-42
    slot = torch.randperm(S + 1, generator=gen, device=DEV)[:S].to(torch.int32)
    kept_rows = torch.full((S, kv_heads, budget), 77, dtype=torch.int32, device=DEV)
    kept_w = torch.full((S + 1, kv_heads, budget + 2), 5.0, device=DEV)
    old = [t.clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    ops.packed_cache_evict(cache, tables, torch.tensor(rows, dtype=torch.int32, device=DEV), w, to, to_tables, kept_rows, budget,
                           keep_first=first, keep_last=last, seq_slot=slot, kept_weights=kept_w, workspace=workspace)
    new = (to.k_codes, to.k_scales, to.v_codes, to.v_scales)
    for s, n in enumerate(rows):
        for h in range(kv_heads):
            mine = w[int(slot[s]), h]
            want = plain.kept(mine[:n].tolist(), budget, first, last)
            assert kept_rows[s, h].tolist() == want + [-1] * (budget - len(want))
            src, at = torch.tensor(want, dtype=torch.long, device=DEV), torch.arange(len(want), device=DEV)
            assert torch.equal(kept_w[int(slot[s]), h, :len(want)].nan_to_num(-3), mine[src].nan_to_num(-3))
            assert (kept_w[int(slot[s]), h, len(want):] == 5).all()
            for a, b in zip(old, new):
                assert torch.equal(a[tables[s].long()[src // page_size], h, src % page_size],
                                   b[to_tables[s].long()[at // to_size], h, at % to_size])
    for a, b in zip(old, (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)):  # what was read stays as it was
        assert torch.equal(a[tables.long().flatten()], b[tables.long().flatten()])


# --------------------------------------------------------------------------------------------- together, refusals
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_request_from_prompt_to_eviction_and_on(ops, workspace, dtype):
    """Write, attend with weights, evict, decode over what stayed: the same as attention over the kept rows alone."""
    heads, kv_heads, D, ps, n, budget = 4, 2, 64, 16, 100, 48
    gen = rng(1)
    qkv = torch.randn(n + 1, (heads + 2 * kv_heads) * D, generator=gen, device=DEV).to(dtype)
    k, v = qkv[:, heads * D:(heads + kv_heads) * D], qkv[:, (heads + kv_heads) * D:]
    cache = ops.PackedPages.empty(20, kv_heads, ps, D, DEV)
    table = torch.arange(7, dtype=torch.int32, device=DEV)[None]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    ops.packed_cache_write(k[:n], v[:n], torch.arange(n, dtype=torch.int32, device=DEV), cache)
    weights, out = torch.rand(1, kv_heads, 128, device=DEV), torch.empty(n, heads * D, dtype=dtype, device=DEV)
    ops.packed_attention(qkv[:n], out, cache, table, i32(0, n), i32(0), n, n, heads, D ** -0.5, weights=weights, workspace=workspace)
    assert abs(float(weights[:, :, :n].sum()) - n * heads) < 1e-3 * n * heads
    kept_rows, kept_weights, to = torch.empty(1, kv_heads, budget, dtype=torch.int32, device=DEV), torch.zeros(1, kv_heads, 128, device=DEV), i32(10, 11, 12, 13)[None]
    ops.packed_cache_evict(cache, table, i32(n), weights, cache, to, kept_rows, budget, keep_first=2, keep_last=10, kept_weights=kept_weights,
                           workspace=workspace)
    ops.packed_cache_write(k[n:], v[n:], i32(13 * ps), cache)
    one = torch.empty(1, heads * D, dtype=dtype, device=DEV)
    ops.packed_attention(qkv[n:], one, cache, to, i32(0, 1), i32(budget), 1, budget + 1, heads, D ** -0.5, weights=kept_weights, workspace=workspace)
    tensors = (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)
    old_k, old_v, _ = plain.request_rows(tensors, table[0], n, ps)
    new_k, new_v, _ = plain.request_rows(tensors, to[0], budget + 1, ps)
    for h in range(kv_heads):
        rows = kept_rows[0, h].long()
        kk, vv = torch.cat([old_k[rows, h], new_k[budget:, h]]), torch.cat([old_v[rows, h], new_v[budget:, h]])
        q = qkv[n:].double()[:, h * 2 * D:(h + 1) * 2 * D].view(1, 2, D)
        want, w, size, _ = plain.attend(q, kk[:, None], vv[:, None], torch.ones(budget + 1, dtype=torch.bool, device=DEV), budget, D ** -0.5)
        got = one[0, h * 2 * D:(h + 1) * 2 * D].double().view(1, 2, D)
        assert ((got - want).abs() <= (size + want.abs() + 4) * (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -16)).all()
        base = torch.cat([weights[0, h][rows], torch.zeros(1, device=DEV)]).double()
        assert ((kept_weights[0, h, :budget + 1].double() - base - w[0]).abs() <= (base + w[0]) * 2.0 ** -14).all()


def test_refusals(ops, workspace):
    from ferrisinfer_b200.errors import KernelError

    cache = ops.PackedPages.empty(4, 2, 16, 64, DEV)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    k, slots = torch.zeros(3, 128, device=DEV), i32(0, 1, 2)
    with pytest.raises(KernelError):
        ops.PackedPages.empty(4, 2, 16, 48, DEV)
    with pytest.raises(KernelError):
        ops.PackedPages.empty(4, 2, 16, 288, DEV)
    with pytest.raises(KernelError):
        ops.PackedPages(cache.k_codes, cache.k_scales[:, :, :, :1], cache.v_codes, cache.v_scales)
    with pytest.raises(KernelError):
        ops.PackedPages(cache.k_codes.float(), cache.k_scales, cache.v_codes, cache.v_scales)
    with pytest.raises(KernelError):
        ops.PackedPages(cache.k_codes.cpu(), cache.k_scales, cache.v_codes, cache.v_scales)
    for call in (lambda: ops.packed_cache_write(k[:2], k, slots, cache), lambda: ops.packed_cache_write(k, k.bfloat16(), slots, cache),
                 lambda: ops.packed_cache_write(k[:, :64], k[:, :64], slots, cache), lambda: ops.packed_cache_write(k, k, slots.long(), cache),
                 lambda: ops.packed_cache_write(k.half(), k.half(), slots, cache), lambda: ops.packed_cache_write(k.cpu(), k.cpu(), slots, cache),
                 lambda: ops.packed_cache_read(cache, slots[:2], k, k), lambda: ops.packed_cache_read(cache, slots, k.t(), k.t())):
        with pytest.raises(KernelError):
            call()
    q = torch.zeros(2, 256, device=DEV, dtype=torch.bfloat16)
    good = dict(q=q, out=torch.zeros_like(q), pages=cache, block_tables=i32(0, 1)[:, None].contiguous(), seq_q_start=i32(0, 1, 2),
                seq_start_row=i32(3, 4), max_q_len=1, max_kv_len=5, num_heads=4, scale=0.1, workspace=workspace)
    ops.packed_attention(**good)
    weights = torch.zeros(2, 2, 5, device=DEV)
    for change in (dict(num_heads=3), dict(out=torch.zeros(2, 128, device=DEV, dtype=torch.bfloat16)), dict(out=torch.zeros(2, 256, device=DEV)),
                   dict(q=q[:, :128]), dict(q=q.half(), out=q.half()), dict(seq_q_start=i32(0, 2)), dict(block_tables=i32(0, 1)),
                   dict(block_tables=i32(0, 1)[:, None].long()), dict(window=-1), dict(max_kv_len=-1), dict(weights=weights[:, :1]),
                   dict(weights=weights[:1]), dict(weights=weights[:, :, :4]), dict(weights=weights.bfloat16()), dict(weights=weights, workspace=None),
                   dict(weights=weights, seq_slot=i32(0)), dict(seq_start_row=i32(3, 4).cpu())):
        with pytest.raises(KernelError):
            ops.packed_attention(**{**good, **change})
    kept_rows = torch.zeros(2, 2, 3, dtype=torch.int32, device=DEV)
    good = dict(pages=cache, block_tables=i32(0, 1)[:, None].contiguous(), seq_rows=i32(5, 5), weights=weights, kept_pages=cache,
                kept_tables=i32(2, 3)[:, None].contiguous(), kept_rows=kept_rows, budget=3, keep_first=1, keep_last=1, workspace=workspace)
    ops.packed_cache_evict(**good)
    other = ops.PackedPages.empty(4, 1, 16, 64, DEV)
    for change in (dict(budget=0), dict(budget=4), dict(keep_first=3), dict(keep_last=-1), dict(kept_pages=other), dict(kept_rows=kept_rows.long()),
                   dict(kept_tables=i32(2, 3)), dict(weights=weights[:1]), dict(seq_rows=i32(5)), dict(kept_weights=weights),
                   dict(kept_weights=torch.zeros(2, 2, 2, device=DEV)), dict(seq_slot=i32(0))):
        with pytest.raises(KernelError):
            ops.packed_cache_evict(**{**good, **change})
    torch.cuda.synchronize()


def test_nothing_to_do(ops, workspace):
    cache = ops.PackedPages.empty(2, 1, 16, 32, DEV)
    none, empty = torch.zeros(0, 32, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV)
    ops.packed_cache_write(none, none, empty, cache)
    ops.packed_cache_read(cache, empty, none, none)
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.packed_attention(none, none, cache, torch.zeros(0, 3, dtype=torch.int32, device=DEV), zero, empty, 0, 0, 1, 1.0, workspace=workspace)
    out = torch.ones(1, 32, device=DEV)
    ops.packed_attention(torch.ones(1, 32, device=DEV), out, cache, torch.zeros(1, 0, dtype=torch.int32, device=DEV),
                         torch.tensor([0, 1], dtype=torch.int32, device=DEV), zero, 1, 0, 1, 1.0, workspace=workspace)
    assert (out == 0).all()
    kept = torch.ones(1, 1, 4, dtype=torch.int32, device=DEV)
    ops.packed_cache_evict(cache, torch.zeros(1, 0, dtype=torch.int32, device=DEV), zero, torch.zeros(1, 1, 0, device=DEV), cache,
                           torch.zeros(1, 0, dtype=torch.int32, device=DEV), kept, 4, workspace=workspace)
    assert (kept == -1).all()
