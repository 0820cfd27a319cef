"""The operators of a step over drafted tokens, as calls of the framework's entry points and in their plain form.

``attend``  queries of trees of drafted tokens (a chain is a tree) attend the paged cache of their requests: every node sees
            the cached text, itself and its ancestors
``probs``   rows of logits become the probabilities that the sampler would draw from (temperature, top-k, top-p)
``verify``  drafted trees are accepted or refused against the target's probabilities with given random numbers: the accepted
            path of every request and the token after it
``keep``    the cached rows of the accepted paths move together behind the text, in every layer

The cache: keys and values [pages, kv heads, page size, head size], a request's row r in page ``tables[r / page size]``.  Node i
of a request with ``start`` rows of text has the row start + i and the position start + its depth.
"""

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def _attend(dtype, seqs, nodes, context, heads, kv_heads, head_dim, ragged=False, chain=False, window=0, page_size=16):
    return {"op": "attend", "dtype": dtype, "seqs": seqs, "nodes": nodes, "context": context, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "ragged": ragged, "chain": chain, "window": window, "page_size": page_size}


def _probs(rows, vocab, temperature, top_k, top_p, mixed=False):
    return {"op": "probs", "rows": rows, "vocab": vocab, "temperature": temperature, "top_k": top_k, "top_p": top_p, "mixed": mixed}


def _verify(seqs, nodes, vocab, drafted, ragged=False, chain=False):
    return {"op": "verify", "seqs": seqs, "nodes": nodes, "vocab": vocab, "drafted": drafted, "ragged": ragged, "chain": chain}


def _keep(dtype, layers, seqs, nodes, accepted, context, kv_heads, head_dim, ragged=False, page_size=16):
    return {"op": "keep", "dtype": dtype, "layers": layers, "seqs": seqs, "nodes": nodes, "accepted": accepted, "context": context,
            "kv_heads": kv_heads, "head_dim": head_dim, "ragged": ragged, "page_size": page_size}


def listed():
    return [
        # one user, four drafted tokens behind the last one: all latency
        dict(_attend("bfloat16", 1, 5, 999, 14, 2, 64, chain=True), name="attend-1"),
        # the benchmark's batch with a tree for each request
        dict(_attend("bfloat16", 8, 16, 4096, 14, 2, 64), name="attend-8"),
        # a busy server: requests at all lengths, small trees of different sizes
        dict(_attend("bfloat16", 64, 8, 4096, 28, 4, 128, ragged=True), name="attend-64"),
        # one user with a very long document and a large tree
        dict(_attend("bfloat16", 1, 64, 131071, 12, 2, 128), name="attend-1-long"),
        # the 32-bit path
        dict(_attend("float32", 6, 13, 1533, 12, 2, 128, ragged=True), name="attend-fp32"),
        # one user's chain of four drafted tokens, sampled as chats are
        dict(_probs(5, 151936, 0.7, 20, 0.9), name="probs-5"),
        # the benchmark's batch, where only the mass decides which tokens stay
        dict(_probs(40, 151936, 0.8, 0, 0.9), name="probs-40-mass"),
        # a busy server's trees, sampled from the whole vocabulary
        dict(_probs(512, 151936, 1.0, 0, 1.0), name="probs-512"),
        # one user's chain, drafted without probabilities (copied from the prompt)
        dict(_verify(1, 5, 151936, False, chain=True), name="verify-1"),
        # a busy server's trees, drawn from a small model's probabilities
        dict(_verify(64, 8, 151936, True), name="verify-64"),
        # one user's accepted tokens in a model of 24 layers
        dict(_keep("bfloat16", 24, 1, 16, 4, 999, 2, 64), name="keep-1"),
        # a busy server's in a model of 28 larger layers
        dict(_keep("bfloat16", 28, 64, 16, 5, 61, 4, 128, ragged=True), name="keep-64"),
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
        what = rng.choice(["attend", "attend", "attend", "attend", "probs", "probs", "verify", "verify", "keep"])
        ragged, chain = rng.random() < 0.5, rng.random() < 0.4
        dtype = "float32" if rng.random() < 0.2 else "bfloat16"
        if what == "attend":
            full = dtype == "float32"
            case = _attend(dtype, between(1, 16 if full else 64), between(1, 24 if full else 64), between(1, 16384 if full else 131071),
                           heads, kv_heads, head_dim, ragged, chain, between(16, 4096) if rng.random() < 0.2 else 0, page_size)
        elif what == "probs":
            temperature, top_k, top_p = rng.choice([(0.7, 20, 0.9), (1.0, 0, 1.0), (0.8, 0, rng.uniform(0.5, 0.99)),
                                                    (rng.uniform(0.3, 1.5), between(2, 1000), 1.0), (0.0, 1, 1.0)])
            case = _probs(between(1, 512), between(1000, 151936), temperature, top_k, top_p, rng.random() < 0.3)
        elif what == "verify":
            case = _verify(between(1, 64), between(1, 64), between(1000, 151936), rng.random() < 0.6, ragged, chain)
            if case["seqs"] * case["nodes"] * case["vocab"] > 64 * 8 * 151936:
                continue
        else:
            nodes = between(3, 64)
            case = _keep(dtype, between(1, 28), between(1, 64), nodes, rng.randint(1, min(8, (nodes - 1) // 2)), between(1, 100),
                         kv_heads, head_dim, ragged, page_size)
            if case["seqs"] * (nodes + case["context"]) * case["layers"] * kv_heads * head_dim > 1.2e8:
                continue
        w = work(case)
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops:
            return case


def _spread(count, most, ragged):
    """``count`` lengths: all ``most``, or from a quarter of it up to it."""
    if not ragged:
        return [most] * count
    return [max(min(most, 1), int(most * (0.25 + 0.75 * ((i + 1) * 0.618034 % 1.0)))) for i in range(count)]


def work(case):
    """Inputs read once, outputs written once; the operations of the formulas."""
    n = case.get("seqs", 0)
    if case["op"] == "probs":  # logits in, probabilities out
        return {"bytes": case["rows"] * (8 * case["vocab"] + 12), "flops": 4 * case["rows"] * case["vocab"]}
    nodes = _spread(n, case["nodes"], case["ragged"])
    if case["op"] == "verify":  # the row that the token after the path comes from, with its draft's; what each node is tried with
        rows = 2 if case["drafted"] else 1
        return {"bytes": n * (4 * case["vocab"] * rows + 4 * case["nodes"] + 8) + sum(nodes) * (12 + 4 * rows),
                "flops": 2 * n * case["vocab"] * rows}
    D, hkv, item = case["head_dim"], case["kv_heads"], 2 if case["dtype"] == "bfloat16" else 4
    if case["op"] == "keep":  # rows read and written
        moved = sum(_spread(n, case["accepted"], case["ragged"]))
        return {"bytes": moved * case["layers"] * 2 * hkv * D * item * 2 + n * 4 * (case["nodes"] + 2), "flops": 0}
    starts, heads, pairs, seen = _spread(n, case["context"], case["ragged"]), case["heads"], 0, 0
    for q, start in zip(nodes, starts):
        text = min(start, case["window"]) if case["window"] else start
        # (a node of a tree has a few ancestors; of a chain, all nodes before it)
        pairs += q * text + (q * (q + 1) // 2 if case["chain"] else int(q * (1 + math.log(q))))
        seen += text + q
    return {"bytes": seen * 2 * hkv * D * item + sum(nodes) * (2 * heads * D * item + 4), "flops": 4 * D * heads * pairs}


# ------------------------------------------------------------------------------------------------ inputs
def _tables(lengths, page_size, rng):
    """Block tables [requests, blocks] that name pages in no order, -1 where a request has none; pages used."""
    blocks = [-(-n // page_size) for n in lengths]
    pages = torch.randperm(sum(blocks), generator=rng, device=DEVICE).to(torch.int32)
    out = torch.full((len(lengths), max(blocks)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, b in enumerate(blocks):
        out[i, :b] = pages[at:at + b]
        at += b
    return out, sum(blocks)


def _parents(nodes, chain, rng):
    """Parents of all requests' nodes: the first is the last known token, the others hang below an earlier one."""
    draws = torch.rand(sum(nodes), generator=rng, device=DEVICE).tolist()
    out = []
    for n in nodes:
        first = len(out)
        out += [i - 1 if chain or i < 2 else int(i * draws[first + i]) for i in range(n)]
    return out


def _starts(nodes):
    return [0] + np.cumsum(nodes).tolist()


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    rng = torch.Generator(device=DEVICE).manual_seed(int(seed))
    state = {"case": case}
    normal = lambda *shape: torch.randn(*shape, generator=rng, device=DEVICE)
    if case["op"] == "probs":
        n, V = case["rows"], case["vocab"]
        logits = normal(n, V) * 2  # most tokens out of the question, a few that could follow
        logits.scatter_(1, torch.randint(V, (n, 20), generator=rng, device=DEVICE), 6 + 2 * normal(n, 20))
        state["logits"], state["out"] = logits, torch.zeros(n, V, device=DEVICE)
        temperature, top_k, top_p = ([case[key]] * n for key in ("temperature", "top_k", "top_p"))
        if case["mixed"]:  # every request has options of its own
            for i in range(1, n):
                temperature[i], top_k[i], top_p[i] = [(0.0, 1, 1.0), (1.0, 0, 1.0), (0.7, 20, 0.9), (0.9, 0, 0.95),
                                                      (case["temperature"], case["top_k"], case["top_p"])][i % 5]
        state["temperature"], state["top_p"] = (torch.tensor(x, dtype=torch.float32, device=DEVICE) for x in (temperature, top_p))
        state["top_k"] = _int32(top_k)
    else:
        nodes = _spread(case["seqs"], case["nodes"], case["ragged"])
        state["q_start"], state["nodes"] = _int32(_starts(nodes)), nodes
    if case["op"] == "verify":
        T, V = sum(nodes), case["vocab"]
        parents = _parents(nodes, case["chain"], rng)
        state["parents"] = _int32(parents)
        state["uniforms"] = torch.rand(T, generator=rng, device=DEVICE)
        logits = normal(T, V)
        if case["drafted"]:
            # the drafting model knows most of what the target knows; every node's children were drawn from its row
            state["draft_probs"] = torch.softmax(3 * logits, -1)
            state["probs"] = torch.softmax(3 * logits + 0.5 * normal(T, V), -1)
            source = state["draft_probs"]
        else:
            state["draft_probs"], state["probs"] = None, torch.softmax(3 * logits, -1)
            source = state["probs"]
        starts = _starts(nodes)
        rows = [first + max(parents[first + i], 0) for first, n in zip(starts, nodes) for i in range(n)]
        # a token of each node's parent's row: where its running sum passes a random number
        sums = torch.cumsum(source, -1)
        want = torch.rand(T, 1, generator=rng, device=DEVICE) * sums[:, -1:][rows]
        state["tokens"] = torch.cat([torch.searchsorted(sums[r:r + 1], want[i:i + 1], right=True) for i, r in enumerate(rows)])
        state["tokens"] = state["tokens"].clamp(max=V - 1).flatten().to(torch.int32)
        state["out_nodes"] = torch.full((case["seqs"], max(nodes)), -1, dtype=torch.int32, device=DEVICE)
        state["out_accepted"], state["out_token"] = (torch.zeros(case["seqs"], dtype=torch.int32, device=DEVICE) for _ in range(2))
    elif case["op"] in ("attend", "keep"):
        D, hkv, ps, dtype = case["head_dim"], case["kv_heads"], case["page_size"], DTYPES[case["dtype"]]
        starts = _spread(case["seqs"], case["context"], case["ragged"])
        state["start_row"], state["starts"] = _int32(starts), starts
        state["tables"], pages = _tables([n + s for n, s in zip(nodes, starts)], ps, rng)
        state["layers"] = []
        for _ in range(case.get("layers", 1)):
            k, v = normal(pages, hkv, ps, D), normal(pages, hkv, ps, D)
            offset = normal(hkv, 1, D) * (torch.rand(hkv, 1, D, generator=rng, device=DEVICE) < 0.06) * 3  # keys have such channels
            state["layers"].append(((k + offset).to(dtype), v.to(dtype)))
        if case["op"] == "attend":
            T = sum(nodes)
            state["parents"] = _int32(_parents(nodes, case["chain"], rng))
            # queries as the fused projection leaves them: the first columns of its rows
            qkv = (normal(T, (case["heads"] + 2 * hkv) * D) * 1.3).to(dtype)
            state["q"], state["out"] = qkv, torch.zeros(T, case["heads"] * D, dtype=dtype, device=DEVICE)
            state["most"] = (max(nodes), max(n + s for n, s in zip(nodes, starts)))
        else:
            # accepted nodes that lie behind the rows they move to, so that a second pass moves the same
            accepted = _spread(case["seqs"], case["accepted"], case["ragged"])
            width = max(nodes)
            path = torch.full((case["seqs"], width), -1, dtype=torch.int32, device=DEVICE)
            path[:, 0] = 0
            for i, (n, a) in enumerate(zip(nodes, accepted)):
                a = accepted[i] = min(a, (n - 1) // 2)
                path[i, 1:a + 1] = (torch.randperm(n - 1 - a, generator=rng, device=DEVICE)[:a].sort().values + a + 1).to(torch.int32)
            state["path"], state["accepted"], state["moves"] = path, _int32(accepted), accepted
    if own:
        from ferrisinfer_b200.engine.workspace import Workspace
        from ferrisinfer_b200.kernels import ops

        state["ops"], state["workspace"] = ops, Workspace(DEVICE)
        if case["op"] == "keep":
            state["cache"] = ops.CacheLayers(state["layers"])
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    return {"attend": _run_attend, "probs": _run_probs, "verify": _run_verify, "keep": _run_keep}[case["op"]](state, case)


def _ancestors(parents):
    """[n, n] truth values: whether node j is node i or above it; depth of every node."""
    n = parents.numel()
    up = parents.long()
    at = torch.arange(n, device=DEVICE)
    seen = torch.eye(n, dtype=torch.bool, device=DEVICE)
    here = at
    for _ in range(n):
        here = torch.where(here >= 0, up[here.clamp(min=0)], here)
        seen |= here[:, None] == at
    return seen, seen.sum(1) - 1


def _run_attend(state, case):
    D, H, hkv, ps, window = case["head_dim"], case["heads"], case["kv_heads"], case["page_size"], case["window"]
    scale, out = D ** -0.5, state["out"]
    k_cache, v_cache = state["layers"][0]
    if own:
        state["ops"].tree_attention(state["q"], out, k_cache, v_cache, state["tables"], state["q_start"], state["start_row"],
                                    state["parents"], state["most"][0], state["most"][1], H, scale, window=window,
                                    workspace=state["workspace"])
        return {"out": out}
    G, at = H // hkv, 0
    for i, (n, start) in enumerate(zip(state["nodes"], state["starts"])):
        row = torch.arange(start + n, device=DEVICE)
        page = state["tables"][i].long()[row // ps]
        k, v = (t[page, :, row % ps].float().permute(1, 0, 2) for t in (k_cache, v_cache))  # [kv heads, rows, D]
        tree, depth = _ancestors(state["parents"][at:at + n])
        sees = torch.cat([torch.ones(n, start, dtype=torch.bool, device=DEVICE), tree], 1)
        if window:
            sees &= torch.cat([row[:start], start + depth]) > (start + depth - window)[:, None]
        q = state["q"][at:at + n, :H * D].float().view(n, hkv, G, D).permute(1, 0, 2, 3).reshape(hkv, n * G, D)
        s = torch.matmul(q, k.transpose(1, 2)) * scale
        s = s.masked_fill(~sees.repeat_interleave(G, 0), float("-inf"))
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
        out[at:at + n] = o.view(hkv, n, G, D).permute(1, 0, 2, 3).reshape(n, H * D).to(out.dtype)
        at += n
    return {"out": out}


def _run_probs(state, case):
    logits, out = state["logits"], state["out"]
    if own:
        state["ops"].sampling_probs(logits, out, state["temperature"], state["top_k"], state["top_p"])
        return {"probs": out}
    n, V = logits.shape
    T, k, p = state["temperature"][:, None], state["top_k"].long()[:, None], state["top_p"][:, None]
    greedy = (T <= 0) | (k == 1) | (p <= 0)
    top = logits.amax(1, keepdim=True)
    if case["mixed"] or case["top_k"] > 0 or case["top_p"] < 1:
        # which tokens stay is a matter of borders: masses in 64 bits
        step = max(1, (1 << 25) // V)
        for a in range(0, n, step):
            b = min(n, a + step)
            values, order = torch.sort(logits[a:b], dim=1, descending=True, stable=True)
            w = torch.exp((values.double() - top[a:b].double()) / T[a:b].double().clamp(min=torch.finfo(torch.float32).eps))
            place = torch.arange(V, device=DEVICE)
            w = torch.where((k[a:b] <= 0) | (place < k[a:b]), w, 0.0)
            before = torch.cumsum(w, 1) - w
            w = torch.where((place == 0) | (p[a:b] >= 1) | (before < p[a:b].double() * w.sum(1, keepdim=True)), w, 0.0)
            w = torch.where(greedy[a:b], (place == 0).double(), w)
            out[a:b].scatter_(1, order, (w / w.sum(1, keepdim=True)).float())
    else:
        if case["temperature"] <= 0:
            out.zero_().scatter_(1, (logits == top).int().argmax(1, keepdim=True), 1.0)
        else:
            torch.sub(logits, top, out=out)
            out.div_(T).exp_()
            out.div_(out.sum(1, keepdim=True))
    return {"probs": out}


def _run_verify(state, case):
    if own:
        state["ops"].verify_tree(state["probs"], state["tokens"], state["parents"], state["q_start"], state["uniforms"], state["out_nodes"],
                                 state["out_accepted"], state["out_token"], draft_probs=state["draft_probs"])
        return {"nodes": state["out_nodes"], "accepted": state["out_accepted"], "token": state["out_token"]}
    parents, tokens, uniforms = (state[x].tolist() for x in ("parents", "tokens", "uniforms"))
    drafted = case["drafted"]
    width, first = state["out_nodes"].shape[1], 0
    for s, n in enumerate(state["nodes"]):
        path = [0]
        while True:
            r, mass = state["probs"][first + path[-1]].double(), 1.0
            q = state["draft_probs"][first + path[-1]].double() if drafted else None
            taken = None
            for c in range(path[-1] + 1, n):
                if parents[first + c] != path[-1] or len(path) == width:
                    continue
                t = tokens[first + c]
                here = r[t].item()
                if uniforms[first + c] * (q[t].item() if drafted else 1.0) * mass < here:
                    taken = c
                    break
                if drafted:
                    left = (r - mass * q).clamp(min=0)
                    total = left.sum().item()
                    if total > 0:
                        r, mass = left, total
                else:
                    mass -= here
                    r = r.clone()
                    r[t] = 0.0
            if taken is None:
                break
            path.append(taken)
        sums = torch.cumsum(r, 0)
        place = torch.searchsorted(sums, uniforms[first] * sums[-1:], right=True)
        last = torch.where(r > 0, torch.arange(r.numel(), device=DEVICE), -1).amax()
        state["out_token"][s] = torch.minimum(place, last)[0].to(torch.int32)
        state["out_accepted"][s] = len(path) - 1
        state["out_nodes"][s] = -1
        state["out_nodes"][s, :len(path)] = _int32(path)
        first += n
    return {"nodes": state["out_nodes"], "accepted": state["out_accepted"], "token": state["out_token"]}


def _run_keep(state, case):
    if own:
        state["ops"].keep_tree_rows(state["cache"], state["tables"], state["start_row"], state["path"], state["accepted"])
        return {"layers": state["layers"]}
    ps, to, src = case["page_size"], [], []
    for i, (start, a) in enumerate(zip(state["starts"], state["moves"])):
        dst = start + 1 + torch.arange(a, device=DEVICE)
        row = start + state["path"][i, 1:a + 1].long()
        table = state["tables"][i].long()
        to.append(table[dst // ps] * ps + dst % ps)
        src.append(table[row // ps] * ps + row % ps)
    to, src = torch.cat(to), torch.cat(src)
    for layer in state["layers"]:
        for t in layer:
            t[to // ps, :, to % ps] = t[src // ps, :, src % ps]
    return {"layers": state["layers"]}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"attend": _exact_attend, "probs": _exact_probs, "verify": _exact_verify, "keep": _exact_keep}[case["op"]](state, case)


def _exact_attend(state, case):
    D, H, ps, window = case["head_dim"], case["heads"], case["page_size"], case["window"]
    out = torch.zeros(state["out"].shape, dtype=torch.float64, device=DEVICE)
    parents, first = state["parents"].tolist(), 0
    for i, (n, start) in enumerate(zip(state["nodes"], state["starts"])):
        # node by node: itself, its parent, its parent's parent ...
        lines = []
        for node in range(n):
            line = [node]
            while parents[first + line[-1]] >= 0:
                line.append(parents[first + line[-1]])
            lines.append(line[:window] if window else line)
        depth = [0] * n
        for node in range(n):
            if parents[first + node] >= 0:
                depth[node] = depth[parents[first + node]] + 1
        sees = torch.zeros(n, start + n, dtype=torch.bool)
        for node, line in enumerate(lines):
            low = max(0, start + depth[node] - window + 1) if window else 0
            sees[node, low:start] = True
            sees[node, [start + x for x in line]] = True
        sees = sees.to(DEVICE)
        row = torch.arange(start + n, device=DEVICE)
        page = state["tables"][i].long()[row // ps]
        for head in range(H):
            kv = head * case["kv_heads"] // H
            k, v = (t[page, kv, row % ps].double() for t in state["layers"][0])
            s = state["q"][first:first + n, head * D:(head + 1) * D].double() @ k.T / math.sqrt(D)
            out[first:first + n, head * D:(head + 1) * D] = torch.softmax(s.masked_fill(~sees, float("-inf")), -1) @ v
        first += n
    return {"out": out}


def _exact_probs(state, case):
    out = torch.zeros(state["out"].shape, dtype=torch.float64, device=DEVICE)
    options = list(zip(*(state[x].tolist() for x in ("temperature", "top_k", "top_p"))))
    for i, (T, k, p) in enumerate(options):
        if T <= 0 or k == 1 or p <= 0:
            out[i, int(np.argmax(state["logits"][i].cpu().numpy()))] = 1.0
        elif k <= 0 and p >= 1:
            out[i] = torch.softmax(state["logits"][i].double() / T, 0)
        else:
            x = state["logits"][i].double().cpu().numpy()
            order = np.argsort(-x, kind="stable")[:k if k > 0 else None]
            w = np.exp((x[order] - x[order[0]]) / T)
            sums = np.cumsum(w)
            if p < 1:
                count = int(np.searchsorted(sums, p * sums[-1], side="left")) + 1
                order, w = order[:count], w[:count]
            out[i, torch.from_numpy(order.copy()).to(DEVICE)] = torch.from_numpy(w / w.sum()).to(DEVICE)
    return {"probs": out}


def _exact_verify(state, case):
    tokens, parents, uniforms = (state[x].cpu().numpy() for x in ("tokens", "parents", "uniforms"))
    nodes = torch.full(state["out_nodes"].shape, -1, dtype=torch.int32)
    accepted, token = [], []
    first = 0
    for s, n in enumerate(state["nodes"]):
        children = {}
        for c in range(1, n):
            children.setdefault(int(parents[first + c]), []).append(c)
        at, path = 0, [0]
        while at is not None:
            p = state["probs"][first + at].cpu().numpy().astype(np.longdouble)
            q = state["draft_probs"][first + at].cpu().numpy().astype(np.longdouble) if case["drafted"] else None
            rest, total, at = p, np.longdouble(1), None  # the target's distribution is rest / total
            for c in children.get(path[-1], []):
                t = tokens[first + c]
                if np.longdouble(uniforms[first + c]) * (q[t] if case["drafted"] else 1) < rest[t] / total:
                    at = c
                    path.append(c)
                    break
                if case["drafted"]:
                    less = np.maximum(rest - total * q, 0)
                    if less.sum() > 0:
                        rest, total = less, less.sum()
                else:
                    total = total - rest[t]
                    rest = np.where(np.arange(rest.size) == t, 0, rest)
        sums = np.cumsum(rest)
        token.append(min(int(np.searchsorted(sums, np.longdouble(uniforms[first]) * sums[-1], side="right")), int(np.nonzero(rest)[0][-1])))
        accepted.append(len(path) - 1)
        nodes[s, :len(path)] = torch.tensor(path, dtype=torch.int32)
        first += n
    return {"nodes": nodes.to(DEVICE), "accepted": _int32(accepted), "token": _int32(token)}


def _exact_keep(state, case):
    ps, layers = case["page_size"], [[t.double() for t in layer] for layer in state["layers"]]
    tables, path = state["tables"].tolist(), state["path"].tolist()
    for i, (start, a) in enumerate(zip(state["starts"], state["moves"])):
        for j in range(1, a + 1):
            src, dst = start + path[i][j], start + j
            for layer in layers:
                for t in layer:
                    t[tables[i][dst // ps], :, dst % ps] = t[tables[i][src // ps], :, src % ps]
    return {"layers": layers}
