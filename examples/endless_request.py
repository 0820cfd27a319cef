"""Attention over requests that never end, in bounded memory: a cache in 4 bits that forgets what attention does not use.

    python examples/endless_request.py [--tokens 4096] [--budget 512]

One layer's queries, keys and values are drawn at random, some keys so that many queries look for them.  The requests bring their
prompts in portions, then single tokens; the cache keeps the rows that attention weighs most.  Printed at the end: rows and bytes
held against a cache that keeps everything in bf16, and how far the last outputs are from attention over everything.
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ferrisinfer_b200.cache.budget import BudgetedCache  # noqa: E402
from ferrisinfer_b200.kernels import ops  # noqa: E402


def main(argv=None) -> dict:
    p = argparse.ArgumentParser()
    p.add_argument("--tokens", type=int, default=4096)
    p.add_argument("--budget", type=int, default=512)
    p.add_argument("--requests", type=int, default=2)
    p.add_argument("--heads", type=int, default=12)
    p.add_argument("--kv-heads", type=int, default=2)
    p.add_argument("--head-dim", type=int, default=128)
    p.add_argument("--portion", type=int, default=256)
    ns = p.parse_args(argv)
    ops.require_device()
    dev, heads, hkv, d = "cuda", ns.heads, ns.kv_heads, ns.head_dim
    gen = torch.Generator(device=dev).manual_seed(0)
    topic = torch.randn(hkv, d, generator=gen, device=dev)  # what queries look for, and one key in a hundred has
    cache = BudgetedCache(ns.requests, hkv, d, ns.budget, slack=128, keep_first=4, keep_last=64, max_portion=ns.portion, device=dev)
    requests = [cache.admit() for _ in range(ns.requests)]
    every_k, every_v = [[] for _ in requests], [[] for _ in requests]
    done, out = 0, None
    while done < ns.tokens:
        n = min(ns.portion, ns.tokens - done) if done < ns.tokens - 64 else 1  # the last 64 tokens one by one
        n = min(n, max(1, ns.tokens - 64 - done))
        T = n * len(requests)
        k = torch.randn(T, hkv, d, generator=gen, device=dev)
        sought = torch.rand(T, 1, 1, generator=gen, device=dev) < 0.01
        k = torch.where(sought, k + 0.6 * topic, k).bfloat16()
        v = torch.randn(T, hkv, d, generator=gen, device=dev).bfloat16()
        q = (torch.randn(T, hkv, heads // hkv, d, generator=gen, device=dev) + topic[:, None]).bfloat16()
        out = torch.empty(T, heads * d, dtype=torch.bfloat16, device=dev)
        cache.step(requests, [n] * len(requests), q.view(T, -1), k.view(T, -1), v.view(T, -1), out, heads, d ** -0.5)
        for i in range(len(requests)):
            every_k[i].append(k[i * n:(i + 1) * n])
            every_v[i].append(v[i * n:(i + 1) * n])
        done += n
    far = []
    for i in range(len(requests)):
        k, v = torch.cat(every_k[i]).float(), torch.cat(every_v[i]).float()
        s = torch.einsum("hgd,nhd->hgn", q[i].float(), k) * d ** -0.5
        full = torch.einsum("hgn,nhd->hgd", torch.softmax(s, -1), v)
        mine = out[i].float().view(hkv, heads // hkv, d)
        far.append(float((mine - full).norm() / full.norm()))
    held = ops.PackedPages.bytes_per_token(hkv, d) * max(cache.rows(r) for r in requests)
    result = {"tokens": done, "rows held": [cache.rows(r) for r in requests], "evictions": cache.evictions, "bytes held": held,
              "bytes of everything in bf16": 4 * hkv * d * done, "last outputs off by": [round(x, 3) for x in far]}
    for key, value in result.items():
        print(f"{key}: {value}")
    return result


if __name__ == "__main__":
    main()
