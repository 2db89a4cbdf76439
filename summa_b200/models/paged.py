"""Paged inference state: sequences of different lengths in one batch, whose keys and values lie in pages of a pool.

`Transformer.make_paged_state` builds it. A slot of the batch is out of use until rows go into it; it takes pages from the pool as its
sequence grows and gives them back when it is released. One page table serves all attention layers, each of which has a pool of its own
(`ops.PagedKV`), in the model's type or in 8 bits. The reference keeps one contiguous cache of one length (`summa-llm/src/generate.rs:127-250`).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Sequence

import torch

from .. import ops
from ..ops.paged import E4M3

PAGE = 64
KINDS = ("paged", "paged_e4m3")


@dataclass
class PagedAttentionState:
    """An attention layer's pages, and the cache that says whose they are."""
    kv: ops.PagedKV
    cache: "PagedCache"


class PagedCache:
    """The page table, the lengths and the free pages of a batch of `batch` slots of up to `capacity` tokens. `num_pages`: pages of the
    pool (as many as all slots at full length need when None)."""

    def __init__(self, batch: int, capacity: int, page: int = PAGE, num_pages: Optional[int] = None, device=None):
        if batch < 1 or capacity < 1:
            raise ValueError(f"a cache of {batch} slots of {capacity} tokens")
        if page not in ops.paged.PAGE_SIZES:
            raise ValueError(f"page size {page}: one of {ops.paged.PAGE_SIZES}")
        self.batch, self.capacity, self.page = batch, capacity, page
        self.per_slot = -(-capacity // page)
        self.num_pages = batch * self.per_slot if num_pages is None else num_pages
        if self.num_pages < 1:
            raise ValueError(f"a pool of {self.num_pages} pages")
        self.table = torch.full((batch, self.per_slot), -1, dtype=torch.int32, device=device)
        self.lengths = torch.full((batch,), -1, dtype=torch.int32, device=device)
        self.held: List[int] = [-1] * batch              # the host's copy of `lengths`
        self.pages: List[List[int]] = [[] for _ in range(batch)]
        self.free = list(range(self.num_pages - 1, -1, -1))
        self.rows: Optional[ops.PagedRows] = None        # of the forward pass under way
        self.fresh: List[int] = []                       # slots that it takes into use, and how many pages it took for each slot
        self.taken = [0] * batch

    def layer(self, kv_heads: int, head_dim: int, dtype: torch.dtype, kind: str) -> PagedAttentionState:
        dev = self.table.device
        shape = (self.num_pages, kv_heads, self.page, head_dim)
        if kind == "paged_e4m3":
            scales = [torch.ones(shape[:2], dtype=torch.float32, device=dev) for _ in range(2)]
            kv = ops.PagedKV(torch.zeros(shape, dtype=E4M3, device=dev), torch.zeros(shape, dtype=E4M3, device=dev), *scales)
        elif kind == "paged":
            kv = ops.PagedKV(torch.zeros(shape, dtype=dtype, device=dev), torch.zeros(shape, dtype=dtype, device=dev))
        else:
            raise ValueError(f"unknown kv_cache `{kind}`: one of {KINDS}")
        return PagedAttentionState(kv, self)

    def active(self) -> List[bool]:
        return [h >= 0 for h in self.held]

    def reserve(self, grow: Sequence[int]) -> List[int]:
        """Pages for `grow[b]` more tokens of each slot (a slot that is not in use begins with them). All of them or, where the pool or
        a slot's capacity does not reach, none. Returns how many each slot took."""
        if len(grow) != self.batch or any(n < 0 for n in grow):
            raise ValueError(f"{list(grow)} more tokens for {self.batch} slots")
        need = []
        for b, n in enumerate(grow):
            end = max(self.held[b], 0) + n
            if n and end > self.capacity:
                raise RuntimeError(f"KV cache overflow: {end} > capacity {self.capacity}")
            need.append(max(0, -(-end // self.page) - len(self.pages[b])) if n else 0)
        if sum(need) > len(self.free):
            raise RuntimeError(f"KV cache overflow: {sum(need)} more pages, and {len(self.free)} of {self.num_pages} are free")
        if not any(need):
            return need
        at, ids = [], []
        for b, n in enumerate(need):
            for _ in range(n):
                at.append(b * self.per_slot + len(self.pages[b]))
                self.pages[b].append(self.free.pop())
                ids.append(self.pages[b][-1])
        dev = self.table.device
        self.table.view(-1)[torch.tensor(at, device=dev)] = torch.tensor(ids, dtype=torch.int32, device=dev)
        return need

    def take(self, grow: Sequence[int]) -> None:
        """`reserve` for a forward pass: `cancel` gives these pages back."""
        self.taken = [a + n for a, n in zip(self.taken, self.reserve(grow))]

    def begin(self, grow: Sequence[int]) -> ops.PagedRows:
        """Describes a forward pass that brings `grow[b]` rows to slot b, and has pages ready for them. It ends with `advance`, or with `cancel`."""
        self.take(grow)
        fresh = [b for b, n in enumerate(grow) if n and self.held[b] < 0]
        self.fresh += fresh
        if fresh:
            self.lengths[torch.tensor(fresh, device=self.lengths.device)] = 0
            for b in fresh:
                self.held[b] = 0
        starts = None
        if any(n != 1 for n in grow):
            at = [0]
            for n in grow:
                at.append(at[-1] + n)
            starts = torch.tensor(at, dtype=torch.int32, device=self.table.device)
        self.rows = ops.PagedRows(self.table, self.lengths, starts, max(max(grow), 1))
        return self.rows

    def begin_step(self, grow: Sequence[int]) -> ops.PagedRows:
        """Describes a step of one row for every slot, of which those that are not in use store nothing."""
        self.take(grow)
        self.rows = ops.PagedRows(self.table, self.lengths)
        return self.rows

    def advance(self, grow: Sequence[int], on_device: bool = True) -> None:
        """The rows of the pass are in the cache. `on_device`: `lengths` too is moved on here."""
        self._close()
        if on_device:
            self.lengths.add_(torch.tensor(list(grow), dtype=torch.int32, device=self.lengths.device))
        self.held = [h + n if n else h for h, n in zip(self.held, grow)]

    def cancel(self) -> None:
        """The pass that was begun did not come to its end: slots have the lengths of before it, those that it took into use are out of it
        again, and the pages that it took are free. (Rows that it has put behind a sequence are not read. In 8 bits they may have raised the
        scale of its last page, and so have rounded that page's codes once more.)"""
        for b, n in reversed(list(enumerate(self.taken))):       # (in the reverse of the order in which they were taken)
            keep = len(self.pages[b]) - n
            if n:
                self.free.extend(reversed(self.pages[b][keep:]))
                del self.pages[b][keep:]
                self.table[b, keep:] = -1
        for b in self.fresh:
            self.held[b] = -1
        self._close()
        self.lengths.copy_(torch.tensor(self.held, dtype=torch.int32))

    def _close(self) -> None:
        self.rows, self.fresh, self.taken = None, [], [0] * self.batch

    def release(self, slot: int) -> None:
        """Takes a slot out of use; its pages go back to the pool."""
        if not 0 <= slot < self.batch:
            raise ValueError(f"slot {slot} of {self.batch}")
        self.free.extend(reversed(self.pages[slot]))
        self.pages[slot], self.taken[slot] = [], 0
        self.fresh = [b for b in self.fresh if b != slot]
        self.held[slot] = -1
        self.lengths[slot] = -1
        self.table[slot] = -1

    def reset(self) -> None:
        for b in range(self.batch):
            if self.held[b] >= 0 or self.pages[b]:
                self.release(b)
