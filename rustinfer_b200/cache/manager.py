"""The cache manager: which pages and which state slot every live request holds.

Layers are sorted into *groups* by what their mixer keeps between steps.  A paged group
(`PagedKV`) has a page pool and a block table per request of its own, so layers that keep
every key and layers that keep a window of them do not share pages; a window group gives
pages back as soon as the window has passed them.  A fixed-state group (`FixedState`)
keeps one row per request slot.  Every request holds one slot while it is live, whether
or not the architecture has fixed state.

Requests can be forked (`fork`): the copies share the pages that are full, whose holders the pool
counts, and own what is still written to (the page the next token goes to, the state slot).  In a
family of equal length every member can take over what another one has (`reorder`), and the pages
that are held can be moved to the lowest numbers (`compact`).  All three say what has to be copied
on the device.

This is host bookkeeping only; the device tensors belong to `CacheStorage`.  In the
reference every layer is full attention over one shared block-id space
(crates/infer-core/src/kv.rs:41-70) and per-request tables are host vectors
(crates/infer-worker/src/application/worker_state.rs:6-24); groups and slots are this
engine's own.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Any, Dict, List, Optional, Sequence, Tuple

from ..parts.base import CacheNeed, FixedState, PagedKV
from .pages import OutOfPages, OutOfSlots, PagePool, StateSlots


@dataclass
class CacheGroup:
    need: CacheNeed
    entries: List[int]                   # run-order entries whose cache lives in this group


@dataclass
class CacheLayout:
    """Run entries sorted into groups; `entry_cache[i]` = (group, index in group), None, or for a
    mixer that declared several needs a list of such pairs in the order of its needs."""
    groups: List[CacheGroup]
    entry_cache: List[Any]
    entry_writes: List[bool]

    @classmethod
    def from_needs(cls, needs: Sequence[Tuple[int, Optional[CacheNeed], Optional[int]]]) -> "CacheLayout":
        groups: List[CacheGroup] = []
        by_need: Dict[CacheNeed, int] = {}
        entry_cache: List[Any] = []
        writes: List[bool] = []

        def place(i: int, need: CacheNeed) -> Tuple[int, int]:
            g = by_need.get(need)
            if g is None:
                g = len(groups)
                by_need[need] = g
                groups.append(CacheGroup(need, []))
            groups[g].entries.append(i)
            return (g, len(groups[g].entries) - 1)

        for i, (_layer, need, cache_of) in enumerate(needs):
            if cache_of is not None:
                entry_cache.append(entry_cache[cache_of])
                writes.append(False)
                continue
            writes.append(True)
            if need is None:
                entry_cache.append(None)
            elif isinstance(need, (tuple, list)):
                entry_cache.append([place(i, n) for n in need])
            else:
                entry_cache.append(place(i, need))
        return cls(groups, entry_cache, writes)

    def paged_groups(self) -> List[int]:
        return [i for i, g in enumerate(self.groups) if isinstance(g.need, PagedKV)]


class Lease:
    """Pages checked out for one step: `commit()` makes them the requests' own (and counts the
    step's tokens), `release()` returns them to the pool and leaves every table as it was
    before.  One of the two must be called; as a context manager the lease commits on a clean
    exit and releases when the body raises.  RustInfer's `KvLease` is the same contract over
    token slots (crates/infer-worker/src/domain/global_kv_alloc.rs:393-461); where its drop of
    an unsettled lease asserts, this one gives the pages back and warns."""

    def __init__(self, manager: "CacheManager", batch: List[Tuple[Any, int]], taken: List[Dict[int, int]]):
        self._m, self._batch, self._taken = manager, batch, taken
        self.settled = False
        manager._leases += 1

    def _settle(self) -> None:
        if self.settled:
            raise RuntimeError("this lease was already committed or released")
        self.settled = True
        self._m._leases -= 1

    def commit(self) -> None:
        self._settle()
        for rid, n in self._batch:
            self._m.commit(rid, n)

    def release(self) -> None:
        self._settle()
        for (rid, _n), taken in zip(self._batch, self._taken):
            r = self._m._req.get(rid)
            if r is None:                                  # closed meanwhile: close() freed its pages
                continue
            for g, k in taken.items():
                if k:
                    table = r.tables[g]
                    self._m.pools[g].free(table[len(table) - k:])
                    del table[len(table) - k:]

    def __enter__(self) -> "Lease":
        return self

    def __exit__(self, exc_type, exc, tb) -> bool:
        if not self.settled:
            if exc_type is None:
                self.commit()
            else:
                self.release()
        return False

    def __del__(self):
        if not getattr(self, "settled", True):
            import warnings
            warnings.warn("a cache lease was dropped unsettled; its pages are given back")
            try:
                self.release()
            except Exception:
                pass


@dataclass
class _Request:
    slot: int
    uid: int = 0                                                  # unique per open(), even if the id returns
    length: int = 0
    tables: Dict[int, List[int]] = field(default_factory=dict)     # group -> page per position block (-1: given back)
    first_live: Dict[int, int] = field(default_factory=dict)       # group -> first block still held
    family: int = 0                                                # uid of the request it was first forked from (its own: none)
    common: int = 1 << 60                                          # any two of a family share at least the lesser of theirs
    changes: int = 0                                               # how often `reorder` has changed the tables
    settled: Dict[int, int] = field(default_factory=dict)          # group -> leading blocks that no `reorder` has changed


@dataclass
class DeviceCopies:
    """What a fork or a reorder has to move on the device.  `pages`: group -> [(source, destination)], the
    first `tokens` tokens of each; `slots`: [(source, destination)]."""
    pages: Dict[int, List[Tuple[int, int]]]
    slots: List[Tuple[int, int]]
    tokens: int


@dataclass
class DeviceReorder:
    """A reorder: entry r of each list takes over what entry parents[r] has.  `pages`: group -> the page every member
    writes to next, of which the first `tokens` tokens are in use (empty where none is)."""
    parents: List[int]
    slots: List[int]
    pages: Dict[int, List[int]]
    tokens: int


class CacheManager:
    def __init__(self, layout: CacheLayout, pages_per_group: Sequence[int], page_size: int,
                 max_requests: int):
        self.layout = layout
        self.page_size = page_size
        self.pools: Dict[int, PagePool] = {}
        paged = layout.paged_groups()
        if len(pages_per_group) != len(paged):
            raise ValueError(f"{len(paged)} paged groups need {len(paged)} pool sizes")
        for g, n in zip(paged, pages_per_group):
            self.pools[g] = PagePool(n)
        self.slots = StateSlots(max_requests)
        self._req: Dict[Any, _Request] = {}
        self._opened = 0
        self._leases = 0                           # leases that are neither committed nor released
        self.newly_opened_slots: List[int] = []    # slots whose fixed state must be zeroed before use

    # ----------------------------------------------------------------- life of a request
    def open(self, request_id: Any) -> int:
        if request_id in self._req:
            raise KeyError(f"request {request_id!r} is already open")
        slot = self.slots.take()
        self._opened += 1
        self._req[request_id] = _Request(slot, self._opened, 0, {g: [] for g in self.pools},
                                         {g: 0 for g in self.pools}, family=self._opened)
        self.newly_opened_slots.append(slot)
        return slot

    def is_open(self, request_id: Any) -> bool:
        return request_id in self._req

    def live_requests(self) -> List[Any]:
        return list(self._req)

    def slot(self, request_id: Any) -> int:
        return self._req[request_id].slot

    def uid(self, request_id: Any) -> int:
        """A number no other open() ever got: tells a request from a later one of the same id."""
        return self._req[request_id].uid

    def length(self, request_id: Any) -> int:
        return self._req[request_id].length

    def close(self, request_id: Any) -> None:
        r = self._req.pop(request_id)
        for g, table in r.tables.items():
            self.pools[g].free(p for p in table if p >= 0)
        self.slots.give_back(r.slot)

    # ------------------------------------------------------------------ forks of a request
    def _no_lease(self, what: str) -> None:
        if self._leases:
            raise RuntimeError(f"{what} while a step's lease is out")

    def fork_needs(self, request_id: Any, copies: int) -> Dict[int, int]:
        """Pages each group hands out for so many forks of a request: its page that is partly filled, once a fork."""
        part = self._req[request_id].length % self.page_size != 0
        return {g: copies if part else 0 for g in self.pools}

    def fork(self, request_id: Any, new_ids: Sequence[Any]) -> DeviceCopies:
        """Opens `new_ids` as copies of a request: they share its full pages and get a page of their own for the one
        that is partly filled, and a state slot.  All or nothing (`OutOfPages`, `OutOfSlots`, KeyError for an id that is
        open)."""
        self._no_lease("fork")
        r = self._req[request_id]
        new_ids = list(new_ids)
        if len(set(new_ids)) != len(new_ids) or any(i in self._req for i in new_ids):
            raise KeyError(f"fork: an id of {new_ids!r} is open already, or stands there twice")
        if len(new_ids) > self.slots.free_count:
            raise OutOfSlots(f"{len(new_ids)} forks, {self.slots.free_count} free request slots")
        for g, k in self.fork_needs(request_id, len(new_ids)).items():
            if k > self.pools[g].free_count:
                raise OutOfPages(k, self.pools[g].free_count, g)
        full, used = divmod(r.length, self.page_size)
        copies = DeviceCopies({g: [] for g in self.pools}, [], used)
        r.common = min(r.common, r.length)
        for i in new_ids:
            slot = self.slots.take()
            self._opened += 1
            tables = {}
            for g, pool in self.pools.items():
                tables[g] = r.tables[g][:full]
                pool.share(p for p in tables[g] if p >= 0)
                if used:
                    (page,) = pool.alloc(1)
                    copies.pages[g].append((r.tables[g][full], page))
                    tables[g].append(page)
            self._req[i] = _Request(slot, self._opened, r.length, tables, dict(r.first_live), family=r.family, common=r.common)
            copies.slots.append((r.slot, slot))
            if r.slot in self.newly_opened_slots:          # nothing in it yet: zeroed like the other one's
                self.newly_opened_slots.append(slot)
        return copies

    def common_length(self, request_ids: Sequence[Any]) -> int:
        """Tokens at the start that these requests certainly share (0 for requests of several families): what their family had when it was forked.
        What a reorder makes them share behind that is not counted."""
        reqs = [self._req[i] for i in request_ids]
        if any(r.family != reqs[0].family for r in reqs):
            return 0
        return min(min(r.common, r.length) for r in reqs)

    def _family(self, request_ids: Sequence[Any], parents: Sequence[int]) -> List[_Request]:
        """The requests of a reorder that can be; raises before anything is changed."""
        reqs = [self._req[i] for i in request_ids]
        if len(parents) != len(reqs) or any(not 0 <= p < len(reqs) for p in parents) or len(set(request_ids)) != len(reqs):
            raise ValueError(f"reorder: {len(reqs)} requests and the parents {list(parents)!r}")
        if any(r.length != reqs[0].length or r.family != reqs[0].family for r in reqs):
            raise ValueError("reorder: the requests are not of one family and one length")
        return reqs

    def reorder_families(self, request_ids: Sequence[Any], parents: Sequence[int], beams: int) -> List[DeviceReorder]:
        """`reorder` of every `beams` requests that follow one another; parents are places in `request_ids`, of the same family.  All
        or nothing: every family is looked at before any is changed."""
        n = len(request_ids)
        if beams < 1 or n % beams or len(parents) != n or len(set(request_ids)) != n:
            raise ValueError(f"reorder: {list(request_ids)!r} and the parents {list(parents)!r} in families of {beams}")
        families = [(request_ids[i: i + beams], [p - i for p in parents[i: i + beams]]) for i in range(0, n, beams)]
        self._no_lease("reorder")
        looked_at = [(self._family(ids, up), up) for ids, up in families]
        return [self._reorder(reqs, up) for reqs, up in looked_at]

    def reorder(self, request_ids: Sequence[Any], parents: Sequence[int]) -> DeviceReorder:
        """Request r takes over what request parents[r] holds, all at once; any mapping.  The requests are of one family and of
        equal length.  Full pages change holders; the page that is partly filled and the state slot stay whose they are, and
        their content moves."""
        self._no_lease("reorder")
        return self._reorder(self._family(request_ids, parents), parents)

    def _reorder(self, reqs: List[_Request], parents: Sequence[int]) -> DeviceReorder:
        full, used = divmod(reqs[0].length, self.page_size) if reqs else (0, 0)
        out = DeviceReorder([int(p) for p in parents], [r.slot for r in reqs], {}, used)
        for g, pool in self.pools.items():
            fresh = []
            for r, p in zip(reqs, parents):
                mine, theirs = r.tables[g], reqs[p].tables[g]
                if mine is theirs:
                    continue
                # pages of tokens that two members have in common are one page: looked at from there on
                b0 = min(r.common, reqs[p].common, reqs[0].length) // self.page_size
                at = next((b for b in range(b0, full) if mine[b] != theirs[b]), full)
                if at < full:
                    fresh.append((r, at, theirs[at:full]))
            for _r, _at, pages in fresh:                   # everyone's new pages before anyone's old ones are given back
                pool.share(p for p in pages if p >= 0)
            for r, at, pages in fresh:
                pool.free(p for p in r.tables[g][at:full] if p >= 0)
                r.tables[g][at:full] = pages
                r.settled[g] = min(at, r.settled.get(g, at))
                r.changes += 1
            out.pages[g] = [r.tables[g][full] for r in reqs] if used else []
        common = [r.common for r in reqs]
        for r, p in zip(reqs, parents):
            r.common = common[p]
        return out

    def changes(self, request_id: Any) -> Tuple[int, Dict[int, int]]:
        """How often the tables were changed other than by new pages, and the leading blocks of each that never were."""
        r = self._req[request_id]
        return r.changes, r.settled

    def compact(self) -> Dict[int, List[Tuple[int, int]]]:
        """Moves the pages that are held to the lowest numbers of their pools: group -> [(from, to)], to be copied on the
        device before anything else is written there."""
        self._no_lease("compact")
        out: Dict[int, List[Tuple[int, int]]] = {}
        for g, pool in self.pools.items():
            moves = pool.compact()
            out[g] = sorted(moves.items())
            if moves:
                for r in self._req.values():
                    table = r.tables[g]
                    hit = [b for b, p in enumerate(table) if p in moves]
                    for b in hit:
                        table[b] = moves[table[b]]
                    if hit:
                        r.settled[g] = min(hit[0], r.settled.get(g, hit[0]))
                        r.changes += 1
        return out

    # -------------------------------------------------------------------------- pages
    def _blocks_for(self, length: int) -> int:
        return (length + self.page_size - 1) // self.page_size

    def pages_needed(self, request_id: Any, new_tokens: int) -> Dict[int, int]:
        """Pages each group must hand out before `new_tokens` more tokens can be stored."""
        r = self._req[request_id]
        want = self._blocks_for(r.length + new_tokens)
        return {g: max(0, want - len(t)) for g, t in r.tables.items()}

    def pages_needed_fresh(self, tokens: int) -> Dict[int, int]:
        """Pages a request that is not open yet would need for its first `tokens` tokens."""
        return {g: self._blocks_for(tokens) for g in self.pools}

    def free_pages(self) -> Dict[int, int]:
        return {g: p.free_count for g, p in self.pools.items()}

    def lease(self, batch: Sequence[Tuple[Any, int]]) -> "Lease":
        """`reserve` as a lease: the pages are checked out for the step and become the requests'
        own when it commits; if the step fails they go back to the pool.  Use as

            with cache.lease(batch):
                run the step            # an exception gives the pages back and passes on
        """
        return Lease(self, list(batch), self.reserve(batch))

    def reserve(self, batch: Sequence[Tuple[Any, int]]) -> List[Dict[int, int]]:
        """Pages for every (request, new tokens) of a step, all or nothing.  Returns, per
        entry of the batch, how many pages each group handed out."""
        total: Dict[int, int] = {g: 0 for g in self.pools}
        per: List[Dict[int, int]] = []
        for rid, n in batch:
            need = self.pages_needed(rid, n)
            per.append(need)
            for g, k in need.items():
                total[g] += k
        for g, k in total.items():
            if k > self.pools[g].free_count:
                raise OutOfPages(k, self.pools[g].free_count, g)
        for (rid, _n), need in zip(batch, per):
            r = self._req[rid]
            for g, k in need.items():
                if k:
                    r.tables[g].extend(self.pools[g].alloc(k))
        return per

    def commit(self, request_id: Any, new_tokens: int) -> None:
        """The step stored `new_tokens` tokens; pages a window has passed are given back."""
        r = self._req[request_id]
        r.length += new_tokens
        if self._blocks_for(r.length) > min((len(t) for t in r.tables.values()), default=1 << 60):
            raise RuntimeError(f"request {request_id!r} committed tokens it holds no pages for")
        for g, table in r.tables.items():
            need = self.layout.groups[g].need
            if need.window is None and need.block is None:
                continue
            # the next token sits at position `length`; pages before the first key it sees (the
            # window's start, or the start of its block of positions) are given back
            keep_from = need.first_key_kept(r.length) // self.page_size
            first = r.first_live[g]
            if keep_from > first:
                self.pools[g].free(table[first:keep_from])
                for b in range(first, keep_from):
                    table[b] = -1
                r.first_live[g] = keep_from

    def block_table(self, request_id: Any, group: int) -> List[int]:
        return self._req[request_id].tables[group]

    def pages_held(self, request_id: Any) -> Dict[int, int]:
        r = self._req[request_id]
        return {g: sum(1 for p in t if p >= 0) for g, t in r.tables.items()}

    # --------------------------------------------------------------------- self-check
    def check_invariants(self) -> None:
        """No page lost, held by more than it counts, written to by two, or both held and free; no slot shared."""
        for g, pool in self.pools.items():
            holders: Dict[int, int] = {}
            for r in self._req.values():
                for b, p in enumerate(r.tables[g]):
                    if p >= 0:
                        holders[p] = holders.get(p, 0) + 1
                        if holders[p] > 1 and (b + 1) * self.page_size > r.length:
                            raise AssertionError(f"group {g}: a page that is written to is held twice")
            if any(pool.holders(p) != n for p, n in holders.items()):
                raise AssertionError(f"group {g}: a page is held by another number than it counts")
            free = pool.free_set()
            if free & set(holders):
                raise AssertionError(f"group {g}: a page is both held and free")
            if len(free) + len(holders) != pool.num_pages:
                raise AssertionError(f"group {g}: {pool.num_pages - len(free) - len(holders)} pages lost")
        slots = [r.slot for r in self._req.values()]
        if len(slots) != len(set(slots)):
            raise AssertionError("a state slot is shared")
        if self.slots.free_count + len(slots) != self.slots.num_slots:
            raise AssertionError("a state slot is lost")
