"""Page and slot allocators: plain host bookkeeping, deterministic.

`PagePool` hands out page ids smallest first and takes them back; handing out is
all-or-nothing.  RustInfer's `GlobalKvAllocator` keeps the same contract over token slots
(sorted free list, smallest ids first, `AllocFull{need, available}`;
crates/infer-worker/src/domain/global_kv_alloc.rs:56-71,129-194).  Where the reference
ignores a double free with a warning, this pool raises: a page freed twice is a fault of
the caller that must not pass silently.

A page may have several holders: requests that were forked from one another share the pages that
are full.  `share` adds a holder, `free` takes one away, and the page is free again when the last
is gone.
"""
from __future__ import annotations

import heapq
from typing import Dict, Iterable, List


class OutOfPages(RuntimeError):
    def __init__(self, need: int, available: int, group: int = 0):
        self.need, self.available, self.group = need, available, group
        super().__init__(f"cache group {group}: {need} pages needed, {available} free")


class OutOfSlots(RuntimeError):
    pass


class PagePool:
    def __init__(self, num_pages: int):
        if num_pages <= 0:
            raise ValueError("a page pool needs at least one page")
        self.num_pages = num_pages
        self._free: List[int] = list(range(num_pages))      # a heap; sorted is a valid heap
        self._holders = [0] * num_pages

    @property
    def free_count(self) -> int:
        return len(self._free)

    def alloc(self, n: int) -> List[int]:
        if n > len(self._free):
            raise OutOfPages(n, len(self._free))
        if n > 8 and n * 16 >= len(self._free):             # a prompt's pages at once: a sorted list is a valid heap and stays one
            self._free.sort()
            out = self._free[:n]
            del self._free[:n]
        else:
            out = [heapq.heappop(self._free) for _ in range(n)]
        for p in out:
            self._holders[p] = 1
        return out

    def share(self, pages: Iterable[int]) -> None:
        """One more holder for each of `pages`, which someone holds."""
        holders = self._holders
        for p in pages:
            if not 0 <= p < self.num_pages or holders[p] == 0:
                raise ValueError(f"page {p} is held by nobody")
            holders[p] += 1

    def free(self, pages: Iterable[int]) -> None:
        free, holders, most = self._free, self._holders, self.num_pages
        for p in pages:
            if not 0 <= p < most:
                raise ValueError(f"page {p} is outside the pool of {self.num_pages}")
            n = holders[p]
            if n == 0:
                raise ValueError(f"page {p} freed twice")
            holders[p] = n - 1
            if n == 1:
                heapq.heappush(free, p)

    def holders(self, page: int) -> int:
        return self._holders[page]

    def compact(self) -> Dict[int, int]:
        """Held pages take the lowest numbers: {old: new} of the ones that move (each to a number that was free)."""
        held = self.num_pages - len(self._free)
        to = sorted(p for p in self._free if p < held)
        moves = dict(zip((p for p in range(held, self.num_pages) if self._holders[p]), to))
        for old, new in moves.items():
            self._holders[new], self._holders[old] = self._holders[old], 0
        self._free = list(range(held, self.num_pages))
        return moves

    def free_set(self) -> set:
        return set(self._free)


class StateSlots:
    """Fixed-size per-request state lives at a slot index a request holds while it is live."""

    def __init__(self, num_slots: int):
        self.num_slots = num_slots
        self._free: List[int] = list(range(num_slots))
        self._held = [False] * num_slots

    @property
    def free_count(self) -> int:
        return len(self._free)

    def take(self) -> int:
        if not self._free:
            raise OutOfSlots(f"all {self.num_slots} request slots are taken")
        s = heapq.heappop(self._free)
        self._held[s] = True
        return s

    def give_back(self, slot: int) -> None:
        if not 0 <= slot < self.num_slots or not self._held[slot]:
            raise ValueError(f"slot {slot} is not held")
        self._held[slot] = False
        heapq.heappush(self._free, slot)
