"""Plain 64-bit forms of the operators of steps over drafted tokens, on the CPU, request by request."""

import math

import torch


def lines_of(parents):
    """Per node: itself, its parent, .. up to the top (what is no earlier node counts as none)."""
    out = []
    for i, up in enumerate(parents):
        out.append([i] + (out[up] if 0 <= up < i else []))
    return out


def tree_attention(q, k_cache, v_cache, tables, q_start, start_row, parents, heads, scale, window=0, max_nodes=256, max_rows=1 << 40):
    """(outputs, sum of p |v|, greatest sum of |q| |k| times the scale of a row) [T, heads x D] in 64 bits; rows that no request brings are NaN."""
    pages, hkv, ps, D = k_cache.shape
    T, G = q.shape[0], heads // hkv
    out = torch.full((T, heads * D), math.nan, dtype=torch.float64)
    mag, size = torch.zeros_like(out), torch.zeros_like(out)
    q = q[:, :heads * D].double().cpu().view(T, heads, D)
    for s, start in enumerate(start_row):
        first, n = q_start[s], min(q_start[s + 1] - q_start[s], max_nodes)
        lines = lines_of(parents[first:first + n])
        rows = [r for r in range(min(start + n, max_rows, len(tables[s]) * ps)) if tables[s][r // ps] >= 0]
        if not rows:
            out[first:first + n] = 0
            continue
        page = torch.tensor([tables[s][r // ps] for r in rows], device=k_cache.device)
        off = torch.tensor([r % ps for r in rows], device=k_cache.device)
        k, v = (t[page, :, off].double().cpu() for t in (k_cache, v_cache))
        at = torch.tensor(rows)
        for i in range(n):
            line = lines[i][:window] if window else lines[i]
            low = max(0, start + len(lines[i]) - window) if window else 0
            sees = ((at >= low) & (at < start)) | torch.isin(at, start + torch.tensor(line))
            for h in range(heads):
                kk, vv = k[sees, h // G], v[sees, h // G]
                if not len(kk):
                    out[first + i, h * D:(h + 1) * D] = 0
                    continue
                p = torch.softmax(kk @ q[first + i, h] * scale, 0)
                here = slice(h * D, (h + 1) * D)
                out[first + i, here] = p @ vv
                mag[first + i, here] = p @ vv.abs()
                size[first + i, here] = (kk.abs() @ q[first + i, h].abs()).max() * abs(scale)
    return out, mag, size


def attention_tolerance(dtype, ref, mag, size, rows, D):
    """How far outputs may be off.  Scores: D products added up in 32 bits, each sum off by 2^-24 of sum |q k| at most, times the scale; a weight
    is then off by as much relative to itself, twice (its sum too).  Weights: exponentials of 2^-22, sums over the rows of 2^-24 each, and where they meet
    bf16 values rounded to bf16 (2^-8).  The output: half a step of its type."""
    score = size * (D + 8) * 2.0 ** -24
    weights = 2 * score + 2.0 ** -21 + rows * 2.0 ** -24 + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0)
    return ref.abs() * torch.finfo(dtype).eps / 2 + mag * weights + 1e-30


def sampling_probs(logits, temperature, top_k, top_p):
    """[n, V] in 64 bits; one temperature, top_k and top_p per row."""
    out = torch.zeros(logits.shape, dtype=torch.float64)
    for r, (row, T, k, p) in enumerate(zip(logits.double().cpu(), temperature, top_k, top_p)):
        row = torch.where(torch.isnan(row), -math.inf, row)
        order = sorted(range(len(row)), key=lambda i, x=row.tolist(): (-x[i], i))
        if not T > 0 or k == 1 or not p > 0:
            out[r, order[0]] = 1
            continue
        top, T = row[order[0]], max(T, torch.finfo(torch.float32).eps)
        w = torch.where(row == top, 1.0, torch.exp((row - top) / T))[order]
        count = len(order) if k <= 0 else min(k, len(order))
        w = w[:count]
        if p < 1:
            reached = torch.nonzero(torch.cumsum(w, 0) >= p * w.sum())
            w = w[:int(reached[0]) + 1] if len(reached) else w
        out[r, order[:len(w)]] = w / w.sum()
    return out


def verify_tree(probs, tokens, parents, q_start, uniforms, width, draft_probs=None):
    """(paths, accepted, next tokens) as lists."""
    clean = lambda t: torch.where(t > 0, t, 0.0).double().cpu()
    probs, draft_probs = clean(probs), None if draft_probs is None else clean(draft_probs)
    V = probs.shape[1]
    paths, accepted, following = [], [], []
    for first, end in zip(q_start[:-1], q_start[1:]):
        n = min(end - first, 256)
        if n <= 0:
            paths.append([-1] * width), accepted.append(0), following.append(-1)
            continue
        path = [0]
        while True:
            x = path[-1]
            r, R, taken = probs[first + x].clone(), 1.0, None
            for c in range(1, n):
                t = tokens[first + c]
                if parents[first + c] != x or c <= x or not 0 <= t < V or len(path) == width:
                    continue
                qt = 1.0 if draft_probs is None else draft_probs[first + x, t].item()
                if uniforms[first + c] * qt * R < r[t].item():
                    taken = c
                    break
                if draft_probs is None:
                    R -= r[t].item()
                    r[t] = 0
                else:
                    left = (r - R * draft_probs[first + x]).clamp(min=0)
                    if left.sum() > 0:
                        r, R = left, left.sum().item()
            if taken is None:
                break
            path.append(taken)
        sums = torch.cumsum(r, 0)
        beyond, some = torch.nonzero(sums > uniforms[first] * sums[-1]), torch.nonzero(r > 0)
        following.append(int(beyond[0]) if len(beyond) else int(some[-1]) if len(some) else -1)
        accepted.append(len(path) - 1)
        paths.append(path + [-1] * (width - len(path)))
    return paths, accepted, following


def keep_tree_rows(caches, tables, start_row, nodes, accepted):
    """Moves the rows of ``caches`` (on the CPU) in place."""
    for s, start in enumerate(start_row):
        rows = {}
        for j in range(1, min(accepted[s], len(nodes[s]) - 1) + 1):
            rows[start + j] = start + nodes[s][j]
        for t in caches:
            ps = t.shape[2]
            held = {dst: t[tables[s][src // ps], :, src % ps].clone() for dst, src in rows.items()}
            for dst, x in held.items():
                t[tables[s][dst // ps], :, dst % ps] = x
