"""The paged cache in 4 bits in plain form: 64-bit arithmetic, one element, row or request at a time, on any device."""

import math

import torch

GROUP = 32


def place(D, keys):
    """Number of the 4-bit place of each element of a head's row: as the bytes of the row are counted, lower half first."""
    out = []
    for d in range(D):
        j, r = divmod(d, GROUP)
        W = D // GROUP
        out.append(((r // 8) * W + j) * 8 + r % 8 if keys else ((r // 4) * W + j) * 4 + r % 4)
    return torch.tensor(out)


def codes_of(rows, keys):
    """uint8 [..., D / 2] as whole numbers [..., D]."""
    D = rows.shape[-1] * 2
    at = place(D, keys).to(rows.device)
    return (rows[..., at // 2].long() >> (4 * (at % 2))) & 15


def pack(codes, keys):
    """The inverse: whole numbers [..., D] as bytes."""
    D = codes.shape[-1]
    at = place(D, keys).to(codes.device)
    halves = torch.empty_like(codes)
    halves[..., at] = codes
    return (halves[..., 0::2] | halves[..., 1::2] << 4).to(torch.uint8)


def values(codes, scales, keys):
    """What packed rows stand for, 64 bits: [..., D]."""
    s = scales.double()
    return codes_of(codes, keys).double() * s[..., 0].repeat_interleave(GROUP, -1) + s[..., 1].repeat_interleave(GROUP, -1)


def scales_of(x):
    """(scale, least) in bf16 of the groups of x [..., D]; NaN where a group is not finite."""
    x = x.double().unflatten(-1, (-1, GROUP))
    low, high = x.amin(-1), x.amax(-1)
    near = low.to(torch.bfloat16)
    least = torch.where(near.double() > low, torch.nextafter(near, torch.full_like(near, -math.inf)), near)
    # (high - least in 32 bits: its rounding may move the scale over a tie between two bf16 numbers)
    scale = ((high.float() - least.float()) / 15).to(torch.bfloat16)
    fine = torch.isfinite(x).all(-1) & torch.isfinite(scale) & torch.isfinite(least)
    return torch.stack([scale, least], -1).masked_fill(~fine[..., None], math.nan)


def cache_of(k, v, page_size, pages=None, spare=0, order=None):
    """Rows k, v [n, kv heads, D] quantised into pages: (four tensors on k's device, page of each block)."""
    n, hkv, D = k.shape
    blocks = -(-n // page_size)
    order = list(range(blocks)) if order is None else order
    total = (max(order) + 1 if order else 1) + spare if pages is None else pages
    out = []
    for x, keys in ((k, True), (v, False)):
        scales = scales_of(x)
        s = scales.double()
        scale, least = s[..., 0].repeat_interleave(GROUP, -1), s[..., 1].repeat_interleave(GROUP, -1)
        codes = ((x.double() - least) / scale).round().clamp(0, 15)
        codes = torch.where(torch.isfinite(codes) & (scale > 0), codes, torch.zeros_like(codes)).long()
        c = torch.full((total, hkv, page_size, D // 2), 0xA7, dtype=torch.uint8, device=k.device)
        t = torch.full((total, hkv, page_size, D // GROUP, 2), math.nan, dtype=torch.bfloat16, device=k.device)
        for r in range(n):
            c[order[r // page_size], :, r % page_size] = pack(codes[r], keys)
            t[order[r // page_size], :, r % page_size] = scales[r]
        out += [c, t]
    return out


def request_rows(cache, table, rows, page_size):
    """Keys and values of rows 0 .. rows - 1 of a request in 64 bits [rows, kv heads, D], and which of them have a page."""
    r = torch.arange(rows, device=cache[0].device)
    table = torch.as_tensor(table, device=cache[0].device).long()
    inside = r // page_size < table.numel()
    page = torch.where(inside, table[(r // page_size).clamp(max=max(table.numel() - 1, 0))], -1)
    at = page.clamp(min=0)
    k = values(cache[0][at, :, r % page_size], cache[1][at, :, r % page_size], True)
    v = values(cache[2][at, :, r % page_size], cache[3][at, :, r % page_size], False)
    return k, v, page >= 0


def attend(q, k, v, has_page, start, scale, window=0):
    """q [n, heads, D] at rows start .. start + n - 1 over k, v [rows, kv heads, D], all 64 bits.  Outputs [n, heads, D], weights
    [kv heads, rows], for each output the sum of the weights times the values' parts without their signs, and for each query
    the greatest sum of |q| |k| of a row that it sees."""
    n, H, D = q.shape
    rows, hkv = k.shape[:2]
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    weights = torch.zeros(hkv, rows, dtype=torch.float64, device=q.device)
    spread = torch.zeros(n, H, dtype=torch.float64, device=q.device)
    j = torch.arange(rows, device=q.device)
    for i in range(n):
        p = start + i
        seen = (j <= p) & has_page
        if window:
            seen &= j > p - window
        at = seen.nonzero()[:, 0]
        if at.numel() == 0:
            continue
        for h in range(H):
            kh, vh = k[at, h * hkv // H], v[at, h * hkv // H]
            s = (kh @ q[i, h]) * scale
            w = torch.softmax(s, 0)
            out[i, h] = w @ vh
            size[i, h] = w @ vh.abs()
            weights[h * hkv // H, at] += w
            spread[i, h] = (kh.abs() @ q[i, h].abs()).max() * abs(scale)
    return out, weights, size, spread


def kept(weights, budget, keep_first, keep_last):
    """Rows that stay of a request and kv head whose rows weigh ``weights`` (a list)."""
    n = len(weights)
    if n <= budget:
        return list(range(n))

    def rank(r):
        if r < keep_first or r >= n - keep_last:
            return (0, 0.0, r)
        w = weights[r]
        return (1, 0.0, r) if math.isnan(w) else (2, -w, r)

    return sorted(sorted(range(n), key=rank)[:budget])
