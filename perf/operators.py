"""The operators of a paged cache in 4 bits, as calls of the framework's entry points and in their plain form.

``write``   keys and values of a step's tokens go into the cache, and are read back as the values it then stands for
``attend``  queries of a step (one token a request, or portions of prompts) attend the cached rows of their requests; with
            ``weights`` every cached row's share of the softmax, summed over the step's queries and the heads that share
            the kv head, comes back too
``evict``   of every request's rows those of the greatest accumulated weight stay, beside its first and last rows, and move
            together into other pages

The cache: ``k_codes`` / ``v_codes`` uint8 [pages, kv heads, page size, head size / 2], ``k_scales`` / ``v_scales`` bf16
[pages, kv heads, page size, head size / 32, 2].  Every 32 neighbours of a head stand as scale * code + least with codes of
0..15; scales hold (scale, least).  In a row of key codes, with W groups of 32, the 4-byte word c W + j (c < 4, j < W) holds
the elements 32 j + 8 c + 0..7, lowest bits first; in a row of value codes the 2-byte word g W + j (g < 8) holds the
elements 32 j + 4 g + 0..3.
"""

import math

import torch

own = False

DEVICE = "cuda"
GROUP = 32
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def _write(dtype, tokens, kv_heads, head_dim, page_size=16):
    return {"op": "write", "dtype": dtype, "tokens": tokens, "kv_heads": kv_heads, "head_dim": head_dim,
            "page_size": page_size}


def _attend(dtype, seqs, q_len, context, heads, kv_heads, head_dim, ragged=False, weights=False, window=0, page_size=16):
    return {"op": "attend", "dtype": dtype, "seqs": seqs, "q_len": q_len, "context": context, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "ragged": ragged, "weights": weights, "window": window,
            "page_size": page_size}


def _evict(seqs, rows, budget, kv_heads, head_dim, ragged=False, page_size=16):
    return {"op": "evict", "dtype": "bfloat16", "seqs": seqs, "rows": rows, "budget": budget, "kv_heads": kv_heads,
            "head_dim": head_dim, "ragged": ragged, "page_size": page_size}


def listed():
    return [
        # the new tokens of a decode step of eight users: all latency
        dict(_write("bfloat16", 8, 2, 64), name="write-step-8"),
        # a batch of prompts at the largest sizes
        dict(_write("bfloat16", 8192, 4, 128), name="write-prompts-8192"),
        # the 32-bit path, an odd number of tokens
        dict(_write("float32", 777, 2, 64), name="write-fp32"),
        # one user's next token in a conversation of medium length
        dict(_attend("bfloat16", 1, 1, 999, 14, 2, 64), name="attend-1"),
        # the benchmark's batch
        dict(_attend("bfloat16", 8, 1, 4096, 14, 2, 64), name="attend-8"),
        # a busy server that will evict: requests at all lengths, weights wanted
        dict(_attend("bfloat16", 64, 1, 4096, 28, 4, 128, ragged=True, weights=True), name="attend-64-weights"),
        # one user with a very long document: what a cache in 4 bits is for
        dict(_attend("bfloat16", 1, 1, 131071, 12, 2, 128), name="attend-1-long"),
        # the 32-bit path's decode step
        dict(_attend("float32", 6, 1, 1533, 12, 2, 128, ragged=True), name="attend-fp32"),
        # short prompts of different lengths that arrive together
        dict(_attend("bfloat16", 6, 700, 0, 12, 2, 128, ragged=True), name="prompts-6"),
        # a portion of a long document whose rows will be evicted by weight
        dict(_attend("bfloat16", 1, 512, 32768, 28, 4, 128, weights=True), name="portion-weights"),
        # one user's conversation outgrows its budget
        dict(_evict(1, 5000, 4096, 2, 64), name="evict-1"),
        # documents of many users are cut down to their budget after the prompt
        dict(_evict(16, 32768, 4096, 4, 128, ragged=True), name="evict-16"),
    ]


def draw(rng):
    def between(lo, hi):  # a whole number, spread over its logarithm
        return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    caps = [work(c) for c in listed()]
    most_bytes, most_flops = max(w["bytes"] for w in caps), max(w["flops"] for w in caps)
    while True:
        heads, kv_heads, head_dim = rng.choice([(14, 2, 64), (12, 2, 128), (28, 4, 128), (16, 4, 128), (16, 16, 64), (24, 2, 64),
                                                (6, 3, 96), (8, 1, 256)])
        page_size = rng.choice([16, 16, 16, 32, 64, 24])
        what = rng.choice(["write", "single", "single", "single", "portion", "portion", "evict"])
        ragged = rng.random() < 0.5
        dtype = "float32" if rng.random() < 0.2 else "bfloat16"
        if what == "write":
            case = _write(dtype, between(1, 8192), kv_heads, head_dim, page_size)
        elif what == "single":
            seqs = between(1, 64)
            case = _attend(dtype, seqs, 1, between(1, 131071), heads, kv_heads, head_dim, ragged, rng.random() < 0.3,
                           between(16, 4096) if rng.random() < 0.2 else 0, page_size)
        elif what == "portion":
            seqs = between(1, 8)
            case = _attend(dtype, seqs, between(2, 2048 if dtype == "bfloat16" else 256), rng.choice([0, between(1, 32768)]), heads,
                           kv_heads, head_dim, ragged, rng.random() < 0.3, between(16, 4096) if rng.random() < 0.2 else 0, page_size)
        else:
            rows = between(64, 65536)
            case = _evict(between(1, 16), rows, between(32, rows), kv_heads, head_dim, ragged, page_size)
        w = work(case)
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops:
            return case


def _spread(count, most, ragged):
    """``count`` lengths: all ``most``, or from a quarter of it up to it."""
    if not ragged:
        return [most] * count
    return [max(min(most, 1), int(most * (0.25 + 0.75 * ((i + 1) * 0.618034 % 1.0)))) for i in range(count)]


def _lengths(case):
    """Per request: (queries of this pass, rows of the cache before them)."""
    n = case["seqs"]
    return list(zip(_spread(n, case["q_len"], case["ragged"]), _spread(n, case["context"], case["ragged"])))


def _visible(q, start, window):
    """Query-row pairs and rows that the queries of one request see."""
    if not window:
        return q * start + q * (q + 1) // 2, start + q
    pairs = sum(min(start + i + 1, window) for i in range(q))
    return pairs, start + q - max(0, start + 1 - window)


def work(case):
    """Inputs read once, outputs written once; the operations of the formulas."""
    D, hkv = case["head_dim"], case["kv_heads"]
    row = 2 * hkv * (D // 2 + 4 * (D // GROUP))  # a token's keys and values in the cache
    item = 2 if case["dtype"] == "bfloat16" else 4
    if case["op"] == "write":  # in, stored, read, out
        values = 2 * hkv * D
        return {"bytes": case["tokens"] * (2 * values * item + 2 * row + 4), "flops": case["tokens"] * values * 8}
    if case["op"] == "evict":  # weights; kept rows out of their pages, into others and read back; their numbers and weights
        rows = _spread(case["seqs"], case["rows"], case["ragged"])
        kept = sum(min(n, case["budget"]) for n in rows)
        return {"bytes": sum(rows) * hkv * 4 + kept * (3 * row + hkv * 8 + 2 * hkv * D * item), "flops": sum(rows) * hkv}
    pairs = seen = tokens = 0
    for q, start in _lengths(case):
        p, r = _visible(q, start, case["window"])
        pairs, seen, tokens = pairs + p, seen + r, tokens + q
    heads = case["heads"]
    return {"bytes": seen * (row + (4 * hkv if case["weights"] else 0)) + 2 * tokens * heads * D * item,
            "flops": 4 * D * heads * pairs}


# ------------------------------------------------------------------------------------------------ inputs
def _quantise(x):
    """Codes (as numbers) and (scale, least) of x [..., D] in groups of 32."""
    x = x.float().unflatten(-1, (-1, GROUP))
    low, high = x.amin(-1), x.amax(-1)
    bits = low.view(torch.int32)  # rounded down to bf16: towards zero by cutting, one further where that went up
    cut = bits & -65536
    least = torch.where((cut != bits) & (bits < 0), cut + 65536, cut).view(torch.float32)
    scale = ((high - least) / 15.0).to(torch.bfloat16).float()
    fine = torch.isfinite(least) & torch.isfinite(scale)
    nan = torch.full_like(least, float("nan"))
    codes = torch.round((x - least[..., None]) / scale[..., None]).clamp(0, 15)
    codes = torch.where((fine & (scale > 0))[..., None], codes, torch.zeros_like(codes))
    scales = torch.stack([torch.where(fine, scale, nan), torch.where(fine, least, nan)], -1).to(torch.bfloat16)
    return codes.to(torch.int32), scales


def _pack(codes, keys):
    """Codes [..., W, 32] as the bytes of a row [..., W * 16]."""
    parts = codes.unflatten(-1, (4, 8) if keys else (8, 4)).transpose(-3, -2).flatten(-3)
    return (parts[..., 0::2] | parts[..., 1::2] << 4).to(torch.uint8)


def _unpack(rows, keys):
    """The inverse of ``_pack``: bytes [..., D / 2] as codes [..., W, 32] in 32 bits."""
    W = rows.shape[-1] * 2 // GROUP
    parts = torch.stack([rows & 15, rows >> 4], -1).flatten(-2)
    return parts.unflatten(-1, (4, W, 8) if keys else (8, W, 4)).transpose(-3, -2).flatten(-2).float()


def _values(codes, scales, keys):
    """What packed rows stand for, in 32 bits: [..., D]."""
    s = scales.float()
    return (_unpack(codes, keys) * s[..., 0:1] + s[..., 1:2]).flatten(-2)


def _cache(pages, kv_heads, page_size, D):
    codes = lambda: torch.zeros(pages, kv_heads, page_size, D // 2, dtype=torch.uint8, device=DEVICE)
    scales = lambda: torch.zeros(pages, kv_heads, page_size, D // GROUP, 2, dtype=torch.bfloat16, device=DEVICE)
    return {"k_codes": codes(), "k_scales": scales(), "v_codes": codes(), "v_scales": scales()}


def _fill(cache, rng):
    """Random keys (with a few channels off zero, as keys have them) and values in every row."""
    pages, kv_heads, page_size, half = cache["k_codes"].shape
    D = 2 * half
    offset = torch.randn(kv_heads, 1, D, generator=rng, device=DEVICE) * (torch.rand(kv_heads, 1, D, generator=rng, device=DEVICE) < 0.06) * 4
    step = max(1, (1 << 24) // (kv_heads * page_size * D))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        for name, keys in (("k", True), ("v", False)):
            x = torch.randn(n, kv_heads, page_size, D, generator=rng, device=DEVICE)
            codes, scales = _quantise(x + offset if keys else x)
            cache[name + "_codes"][p:p + n] = _pack(codes, keys)
            cache[name + "_scales"][p:p + n] = scales


def _tables(lengths, page_size, rng, first=0):
    """Block tables [requests, blocks] that name pages in no order, -1 where a request has none; pages used."""
    blocks = [-(-n // page_size) for n in lengths]
    pages = torch.randperm(sum(blocks), generator=rng, device=DEVICE).to(torch.int32) + first
    out = torch.full((len(lengths), max(blocks)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, b in enumerate(blocks):
        out[i, :b] = pages[at:at + b]
        at += b
    return out, sum(blocks)


def prepare(case, seed):
    rng = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype, D, hkv, ps = DTYPES[case["dtype"]], case["head_dim"], case["kv_heads"], case["page_size"]
    state = {"case": case}
    if case["op"] == "write":
        T = case["tokens"]
        pages = -(-T // ps) + 1
        # keys and values as the fused projection leaves them: columns of one matrix, behind the queries
        qkv = torch.randn(T, 4 * hkv * D, generator=rng, device=DEVICE) * 2
        qkv[:, ::29] *= 6
        qkv = qkv.to(dtype)
        state["k"], state["v"] = qkv[:, 2 * hkv * D:3 * hkv * D], qkv[:, 3 * hkv * D:]
        state["slots"] = torch.randperm(pages * ps, generator=rng, device=DEVICE)[:T].to(torch.int32)
        state["cache"] = _cache(pages, hkv, ps, D)
        state["k_out"], state["v_out"] = (torch.zeros(T, hkv * D, dtype=dtype, device=DEVICE) for _ in range(2))
    elif case["op"] == "attend":
        lengths = _lengths(case)
        state["tables"], pages = _tables([q + s for q, s in lengths], ps, rng)
        state["cache"] = _cache(pages, hkv, ps, D)
        _fill(state["cache"], rng)
        starts = [0]
        for q, _ in lengths:
            starts.append(starts[-1] + q)
        state["q_start"] = torch.tensor(starts, dtype=torch.int32, device=DEVICE)
        state["start_row"] = torch.tensor([s for _, s in lengths], dtype=torch.int32, device=DEVICE)
        state["lengths"] = lengths
        state["q"] = (torch.randn(starts[-1], case["heads"] * D, generator=rng, device=DEVICE) * 1.3).to(dtype)
        state["out"] = torch.zeros_like(state["q"])
        most = max(q + s for q, s in lengths)
        state["weights"] = torch.zeros(case["seqs"], hkv, most, device=DEVICE) if case["weights"] else None
        state["most"] = (max(q for q, _ in lengths), most)
    else:
        rows = _spread(case["seqs"], case["rows"], case["ragged"])
        budget = min(case["budget"], max(rows))
        state["tables"], pages = _tables(rows, ps, rng)
        kept = [min(n, budget) for n in rows]
        state["kept_tables"], more = _tables(kept, ps, rng, first=pages)
        state["cache"] = _cache(pages + more, hkv, ps, D)
        _fill(state["cache"], rng)
        state["rows"] = torch.tensor(rows, dtype=torch.int32, device=DEVICE)
        # weights as attention leaves them: most rows next to nothing, a few a lot, many exactly alike
        w = torch.rand(case["seqs"], hkv, max(rows), generator=rng, device=DEVICE)
        state["weights"] = torch.where(w < 0.3, torch.round(w * 40) / 4096, 0.01 / (1.0001 - w) ** 1.5)
        state["kept_weights"] = torch.zeros(case["seqs"], hkv, budget, device=DEVICE)
        state["kept_rows"] = torch.full((case["seqs"], hkv, budget), -1, dtype=torch.int32, device=DEVICE)
        at = torch.arange(budget, device=DEVICE)
        slots = state["kept_tables"].long()[:, at // ps] * ps + at % ps
        state["slots"] = torch.where(at < torch.tensor(kept, device=DEVICE)[:, None], slots, -1).to(torch.int32).flatten()
        state["k_out"], state["v_out"] = (torch.zeros(case["seqs"] * budget, hkv * D, dtype=dtype, device=DEVICE) for _ in range(2))
        state["budget"] = budget
        state["keep"] = (min(4, budget // 4), budget // 4)  # first and last rows that stay whatever their weight
        state["lengths"] = rows
    if own:
        from ferrisinfer_b200.engine.workspace import Workspace
        from ferrisinfer_b200.kernels import ops

        state["ops"], state["pages"], state["workspace"] = ops, ops.PackedPages(**state["cache"]), Workspace(DEVICE)
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    return {"write": _run_write, "attend": _run_attend, "evict": _run_evict}[case["op"]](state, case)


def _read(cache, slots, dtype):
    """Keys and values at the slots (nothing at -1), [n, kv heads * D]."""
    ps = cache["k_codes"].shape[2]
    at = slots.long().clamp(min=0)
    out = []
    for name, keys in (("k", True), ("v", False)):
        x = _values(cache[name + "_codes"][at // ps, :, at % ps], cache[name + "_scales"][at // ps, :, at % ps], keys)
        out.append(torch.where((slots >= 0)[:, None], x.flatten(1), torch.zeros((), device=DEVICE)).to(dtype))
    return out


def _run_write(state, case):
    if own:
        ops = state["ops"]
        ops.packed_cache_write(state["k"], state["v"], state["slots"], state["pages"])
        ops.packed_cache_read(state["pages"], state["slots"], state["k_out"], state["v_out"])
        return {"k": state["k_out"], "v": state["v_out"]}
    cache, at, ps = state["cache"], state["slots"].long(), case["page_size"]
    for name, keys in (("k", True), ("v", False)):
        codes, scales = _quantise(state[name].unflatten(-1, (case["kv_heads"], -1)))
        cache[name + "_codes"][at // ps, :, at % ps] = _pack(codes, keys)
        cache[name + "_scales"][at // ps, :, at % ps] = scales
    k, v = _read(cache, state["slots"], state["k"].dtype)
    return {"k": k, "v": v}


def _softmax_rows(qg, k, v, visible, scale):
    """qg [B, Hkv, R, D], k and v [B, L, Hkv, D], visible [B, R, L]: outputs [B, Hkv, R, D], weights [B, Hkv, L]."""
    s = torch.matmul(qg, k.permute(0, 2, 3, 1)) * scale
    s = torch.where(visible[:, None], s, torch.full((), float("-inf"), device=DEVICE))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isfinite(top), top, torch.zeros((), device=DEVICE)))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones((), device=DEVICE))
    return torch.matmul(p, v.permute(0, 2, 1, 3)), p.sum(-2)


def _run_attend(state, case):
    D, H, hkv, ps, window = case["head_dim"], case["heads"], case["kv_heads"], case["page_size"], case["window"]
    scale = D ** -0.5
    if own:
        state["ops"].packed_attention(state["q"], state["out"], state["pages"], state["tables"], state["q_start"],
                                      state["start_row"], state["most"][0], state["most"][1], H, scale, window=window,
                                      weights=state["weights"], add_weights=False, workspace=state["workspace"])
        return {"out": state["out"], "weights": state["weights"]} if case["weights"] else {"out": state["out"]}
    cache, G = state["cache"], H // hkv
    out, weights = state["out"], state["weights"]

    def gather(tables, length):
        at = torch.arange(length, device=DEVICE)
        pages = tables.long().clamp(min=0)[:, at // ps]  # [B, length]
        return [_values(cache[n + "_codes"][pages, :, at % ps], cache[n + "_scales"][pages, :, at % ps], n == "k") for n in "kv"]

    if state["most"][0] == 1:  # one token a request: requests side by side, few enough at once
        B, L = case["seqs"], state["most"][1]
        step = max(1, (1 << 28) // (L * hkv * D))
        for b in range(0, B, step):
            m = min(step, B - b)
            k, v = gather(state["tables"][b:b + m], L)
            row, j = state["start_row"][b:b + m, None, None], torch.arange(L, device=DEVICE)
            visible = (j <= row) & ((j > row - window) if window else True)
            o, w = _softmax_rows(state["q"][b:b + m].float().view(m, hkv, G, D), k, v, visible, scale)
            out[b:b + m] = o.reshape(m, H * D).to(out.dtype)
            if weights is not None:
                weights[b:b + m] = w
    else:
        at = 0
        for i, (n, start) in enumerate(state["lengths"]):
            L = n + start
            k, v = gather(state["tables"][i:i + 1], L)
            row, j = start + torch.arange(n, device=DEVICE)[:, None], torch.arange(L, device=DEVICE)
            visible = ((j <= row) & ((j > row - window) if window else True)).repeat_interleave(G, 0)[None]
            qg = state["q"][at:at + n].float().view(n, hkv, G, D).transpose(0, 1).reshape(1, hkv, n * G, D)
            o, w = _softmax_rows(qg, k, v, visible, scale)
            out[at:at + n] = o.view(hkv, n, G, D).transpose(0, 1).reshape(n, H * D).to(out.dtype)
            if weights is not None:
                weights[i, :, :L] = w[0]
            at += n
    return {"out": out, "weights": weights} if case["weights"] else {"out": out}


def _run_evict(state, case):
    first, last = state["keep"]
    budget, hkv, ps = state["budget"], case["kv_heads"], case["page_size"]
    if own:
        ops = state["ops"]
        ops.packed_cache_evict(state["pages"], state["tables"], state["rows"], state["weights"], state["pages"],
                               state["kept_tables"], state["kept_rows"], budget, keep_first=first, keep_last=last,
                               kept_weights=state["kept_weights"], workspace=state["workspace"])
        ops.packed_cache_read(state["pages"], state["slots"], state["k_out"], state["v_out"])
        return {"rows": state["kept_rows"], "weights": state["kept_weights"], "k": state["k_out"], "v": state["v_out"]}
    cache, heads = state["cache"], torch.arange(hkv, device=DEVICE)[:, None]
    for i, n in enumerate(state["lengths"]):
        w = state["weights"][i, :, :n]
        if n > budget:
            rank = w.clone()
            rank[:, :first] = float("inf")
            rank[:, n - last:] = float("inf")
            rows = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :budget].sort(1).values
        else:
            rows = torch.arange(n, device=DEVICE).expand(hkv, n)
        m = rows.shape[1]
        to = torch.arange(m, device=DEVICE)
        src, dst = state["tables"][i].long()[rows // ps], state["kept_tables"][i].long()[to // ps].expand(hkv, m)
        for t in cache.values():
            t[dst, heads, (to % ps).expand(hkv, m)] = t[src, heads, rows % ps]
        state["kept_rows"][i, :, :m] = rows.to(torch.int32)
        state["kept_weights"][i, :, :m] = torch.gather(w, 1, rows)
    k, v = _read(cache, state["slots"], state["k_out"].dtype)
    return {"rows": state["kept_rows"], "weights": state["kept_weights"], "k": k, "v": v}


# ------------------------------------------------------------------------------------------------ 64 bits
def _row64(cache, name, page, head, off):
    """Rows (page, head, off: index tensors) of the keys or values in 64 bits, element by element from their places."""
    codes, scales = cache[name + "_codes"][page, head, off], cache[name + "_scales"][page, head, off].double()
    D = codes.shape[-1] * 2
    W, d = D // GROUP, torch.arange(D, device=DEVICE)
    j, r = d // 32, d % 32
    nibble = ((r // 8) * W + j) * 8 + r % 8 if name == "k" else ((r // 4) * W + j) * 4 + r % 4
    code = (codes[..., nibble // 2].long() >> (4 * (nibble % 2))) & 15
    return code.double() * scales[..., j, 0] + scales[..., j, 1]


def exact(case, seed):
    state = prepare(case, seed)
    cache, D, hkv, ps = state["cache"], case["head_dim"], case["kv_heads"], case["page_size"]
    if case["op"] == "write":
        outs = {}
        for name in "kv":
            x = state[name].double().reshape(case["tokens"], hkv * D // 32, 32)
            low = x.min(-1).values
            near = low.to(torch.bfloat16)  # the nearest number of 8 bits, or the one below it
            less = torch.nextafter(near, torch.full_like(near, float("-inf")))
            least = torch.where(near.double() > low, less, near).double()
            scale = ((x.max(-1).values - least) / 15).to(torch.bfloat16).double()
            code = ((x - least[..., None]) / scale[..., None]).round().clamp(0, 15)
            outs[name] = (code * scale[..., None] + least[..., None]).reshape(case["tokens"], hkv * D)
        return outs
    if case["op"] == "evict":
        if sum(state["lengths"]) * hkv > 6e6:
            return None
        first, last = state["keep"]
        budget = state["budget"]
        kept_weights = torch.zeros(case["seqs"], hkv, budget, dtype=torch.float64, device=DEVICE)
        k, v = (torch.zeros(case["seqs"], budget, hkv, D, dtype=torch.float64, device=DEVICE) for _ in range(2))
        for i, n in enumerate(state["lengths"]):
            at = torch.arange(n, device=DEVICE)
            for h in range(hkv):
                w = state["weights"][i, h, :n].double()
                key = torch.where((at < first) | (at >= n - last), float("inf"), w)
                order = sorted(range(n), key=lambda r, key=key.tolist(): (-key[r], r))[:budget] if n > budget else range(n)
                rows = torch.tensor(sorted(order), device=DEVICE)
                kept_weights[i, h, :len(rows)] = w[rows]
                page = state["tables"][i].long()[rows // ps]
                k[i, :len(rows), h] = _row64(cache, "k", page, h, rows % ps)
                v[i, :len(rows), h] = _row64(cache, "v", page, h, rows % ps)
        return {"rows": None, "weights": kept_weights, "k": k.flatten(0, 1).flatten(1), "v": v.flatten(0, 1).flatten(1)}
    H, window = case["heads"], case["window"]
    if work(case)["flops"] > 4e11:
        return None
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device=DEVICE)
    weights = torch.zeros(case["seqs"], hkv, state["most"][1], dtype=torch.float64, device=DEVICE)
    at = 0
    for i, (n, start) in enumerate(state["lengths"]):
        j = torch.arange(start + n, device=DEVICE)
        page = state["tables"][i].long()[j // ps]
        for h in range(hkv):
            k, v = _row64(cache, "k", page, h, j % ps), _row64(cache, "v", page, h, j % ps)
            for head in range(h * (H // hkv), (h + 1) * (H // hkv)):
                q = state["q"][at:at + n, head * D:(head + 1) * D].double()
                s = q @ k.T / math.sqrt(D)
                p = start + torch.arange(n, device=DEVICE)[:, None]
                s.masked_fill_((j > p) | ((j <= p - window) if window else torch.zeros((), dtype=torch.bool, device=DEVICE)), float("-inf"))
                s = torch.softmax(s, -1)
                out[at:at + n, head * D:(head + 1) * D] = s @ v
                weights[i, h, :start + n] += s.sum(0)
        at += n
    return {"out": out, "weights": weights} if case["weights"] else {"out": out}
