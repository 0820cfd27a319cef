"""Keys and values of one attention layer for several requests, in 4 bits and within a budget of rows.

A request may run for ever in bounded memory: every step's attention adds to each cached row's accumulated weight, and
when a request has outgrown its budget by ``slack`` rows, each kv head keeps its first ``keep_first`` rows, its
last ``keep_last`` and, of the others, those that attention has weighed most (the lower row first among equals).  The rows that
stay move into fresh pages and the old pages go back to the pool.  The layer's keys are expected as they are attended
(rotated by their own positions), so rows may stand anywhere; a window over positions does not go with it.

The engine's own cache manager counts a row for every token of a request and shares prompts' pages between requests;
this class is for callers that drive ``ops.packed_attention`` themselves.
"""

from __future__ import annotations

from typing import Sequence

import numpy as np
import torch

from ..engine.workspace import Workspace
from ..errors import CacheError
from ..kernels import ops
from .pages import PagePool


class BudgetedCache:
    def __init__(self, max_requests: int, kv_heads: int, head_dim: int, budget: int, slack: int = 256, keep_first: int = 4,
                 keep_last: int = 64, max_portion: int = 512, page_size: int = 16, device="cuda"):
        """``budget`` rows per request and kv head after an eviction; before the next one there may be up to ``slack`` more.
        ``max_portion``: the most tokens that a request brings in one step."""
        if max_requests <= 0 or page_size <= 0 or max_portion <= 0 or slack < 0:
            raise CacheError(f"{max_requests} requests, pages of {page_size} rows, portions of {max_portion}, slack of {slack}")
        if budget <= 0 or keep_first < 0 or keep_last < 0 or keep_first + keep_last > budget:
            raise CacheError(f"{keep_first} first and {keep_last} last rows of a budget of {budget}")
        self.budget, self.slack, self.keep_first, self.keep_last = int(budget), int(slack), int(keep_first), int(keep_last)
        self.page_size, self.max_portion = int(page_size), int(max_portion)
        self.device = torch.device(device)
        self.max_rows = self.budget + self.slack + self.max_portion
        # every request at its most, and the rows that stay of one request beside the pages that they leave
        self.pool = PagePool(max_requests * self._blocks(self.max_rows) + self._blocks(self.budget))
        self.pages = ops.PackedPages.empty(self.pool.num_pages, kv_heads, page_size, head_dim, self.device)
        # two sets: an eviction takes a request's weights from one into the other
        self._weights = torch.zeros(2, max_requests, kv_heads, self.max_rows, dtype=torch.float32, device=self.device)
        self._set = [0] * max_requests
        self._rows = [0] * max_requests  # rows that each request holds
        self._tables: list = [[] for _ in range(max_requests)]
        self._held = [False] * max_requests
        self.workspace = Workspace(self.device)
        self.evictions = 0
        self.last_kept: dict = {}  # request -> int32 [kv heads, budget]: rows that stayed at its last eviction

    def _blocks(self, rows: int) -> int:
        return -(-rows // self.page_size)

    # ------------------------------------------------------------------ requests
    def admit(self) -> int:
        """A request's number; its cache is empty."""
        for r, held in enumerate(self._held):
            if not held:
                self._held[r], self._rows[r], self._tables[r] = True, 0, []
                self.last_kept.pop(r, None)
                return r
        raise CacheError(f"all {len(self._held)} requests are taken")

    def release(self, request: int) -> None:
        self._check(request)
        for page in self._tables[request]:
            self.pool.release(page)
        self._held[request], self._rows[request], self._tables[request] = False, 0, []

    def rows(self, request: int) -> int:
        self._check(request)
        return self._rows[request]

    def weights(self, request: int) -> torch.Tensor:
        """Accumulated weight of the request's rows, fp32 [kv heads, rows]."""
        self._check(request)
        return self._weights[self._set[request], request, :, :self._rows[request]]

    def table(self, request: int) -> list:
        """Pages of the request's rows, in order."""
        self._check(request)
        return list(self._tables[request])

    def _check(self, request: int) -> None:
        if not (0 <= request < len(self._held)) or not self._held[request]:
            raise CacheError(f"request {request} is not admitted")

    # ---------------------------------------------------------------------- steps
    def _device_ints(self, *arrays) -> list:
        """The arrays as int32 tensors on the device, with one copy."""
        flat = np.concatenate([np.asarray(a, dtype=np.int32).reshape(-1) for a in arrays])
        dev = torch.from_numpy(flat).to(self.device)
        out, at = [], 0
        for a in arrays:
            a = np.asarray(a)
            out.append(dev[at:at + a.size].view(a.shape))
            at += a.size
        return out

    def _table_array(self, tables: Sequence[list]):
        out = np.full((len(tables), max(1, max(len(t) for t in tables))), -1, dtype=np.int32)
        for i, t in enumerate(tables):
            out[i, :len(t)] = t
        return out

    def step(self, requests: Sequence[int], q_lens: Sequence[int], q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
             num_heads: int, scale: float) -> None:
        """One step of the layer: request ``requests[i]`` brings ``q_lens[i]`` consecutive rows of ``q``, ``k``, ``v`` (columns of a fused
        projection will do, as in ``ops.packed_attention``); their keys and values enter the cache, their queries attend it into
        ``out``, and requests that have outgrown budget and slack are cut down."""
        if not requests or len(requests) != len(q_lens) or len(set(requests)) != len(requests):
            raise CacheError(f"a step of {len(requests)} requests with {len(q_lens)} lengths")
        if sum(q_lens) != q.shape[0] or any(not 0 < n <= self.max_portion for n in q_lens):
            raise CacheError(f"portions of {list(q_lens)} tokens (at most {self.max_portion} each) for {q.shape[0]} rows")
        for r in requests:
            self._check(r)
        starts, slots = [0], []
        for r, n in zip(requests, q_lens):
            table, rows = self._tables[r], self._rows[r]
            missing = self._blocks(rows + n) - len(table)
            if missing > 0:
                table.extend(self.pool.alloc(missing))
            at = np.arange(rows, rows + n)
            slots.append(np.asarray(table, dtype=np.int64)[at // self.page_size] * self.page_size + at % self.page_size)
            starts.append(starts[-1] + n)
        slot_mapping, tables, q_start, start_row, places = self._device_ints(
            np.concatenate(slots), self._table_array([self._tables[r] for r in requests]), starts, [self._rows[r] for r in requests],
            [self._set[r] * len(self._held) + r for r in requests])
        ops.packed_cache_write(k, v, slot_mapping, self.pages)
        ops.packed_attention(q, out, self.pages, tables, q_start, start_row, max(q_lens), max(self._rows[r] + n for r, n in zip(requests, q_lens)),
                             num_heads, scale, weights=self._weights.flatten(0, 1), seq_slot=places, workspace=self.workspace)
        for r, n in zip(requests, q_lens):
            self._rows[r] += n
        for r in requests:  # one at a time: the pool has fresh pages for one
            if self._rows[r] > self.budget + self.slack:
                self.evict(r)

    def evict(self, request: int) -> None:
        """Cut the request down to its budget now (nothing happens within it)."""
        self._check(request)
        n = self._rows[request]
        if n <= self.budget:
            return
        fresh = self.pool.alloc(self._blocks(self.budget))
        tables, to, rows = self._device_ints(np.asarray([self._tables[request]]), np.asarray([fresh]), [n])
        kept = torch.empty(1, self.pages.kv_heads, self.budget, dtype=torch.int32, device=self.device)
        here = self._set[request]
        ops.packed_cache_evict(self.pages, tables, rows, self._weights[here, request:request + 1], self.pages, to, kept, self.budget,
                               keep_first=self.keep_first, keep_last=self.keep_last,
                               kept_weights=self._weights[1 - here, request:request + 1], workspace=self.workspace)
        for page in self._tables[request]:  # (whoever gets them next writes behind this on the stream)
            self.pool.release(page)
        self._tables[request], self._rows[request], self._set[request] = fresh, self.budget, 1 - here
        self.last_kept[request] = kept[0]
        self.evictions += 1
