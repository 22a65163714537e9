"""Forks, reorders and compaction in the cache manager, and a beam search's own bookkeeping, on the host."""
import random

import numpy as np
import pytest

from rustinfer_b200.cache.manager import CacheLayout, CacheManager
from rustinfer_b200.cache.pages import OutOfPages, OutOfSlots, PagePool
from rustinfer_b200.engine.beam import BeamParams, _Search, take_rows
from rustinfer_b200.parts.base import FixedState, PagedKV

PAGE = 4
FULL, WIN, BLOCK, STATE = PagedKV(2, 16, None), PagedKV(2, 16, 11), PagedKV(2, 16, None, block=6), FixedState((8,), "float32")


def manager(pages, requests, *needs):
    lay = CacheLayout.from_needs([(i, n, None) for i, n in enumerate(needs)])
    return CacheManager(lay, [pages] * len(lay.paged_groups()), PAGE, requests)


def test_pages_with_several_holders():
    p = PagePool(6)
    a = p.alloc(3)
    p.share([a[0], a[1]])
    p.share([a[0]])
    p.free(a)
    assert p.free_count == 4 and p.holders(a[0]) == 2 and p.holders(a[2]) == 0
    with pytest.raises(ValueError, match="nobody"):
        p.share([a[2]])
    with pytest.raises(ValueError, match="nobody"):
        p.share([7])
    p.free([a[0]]); p.free([a[0], a[1]])
    assert p.free_count == 6
    with pytest.raises(ValueError, match="twice"):
        p.free([a[0]])


def test_compacting_a_pool():
    p = PagePool(10)
    p.alloc(9)
    p.share([8])
    p.free([0, 2, 3, 5, 6])
    assert p.compact() == {4: 0, 7: 2, 8: 3}
    assert p.free_set() == set(range(4, 10)) and p.holders(3) == 2 and p.compact() == {}
    assert p.alloc(1) == [4]


class Device:
    """What the pages and slots of a manager hold, moved as the manager says."""

    def __init__(self, m):
        self.m = m
        self.pages = {g: [[None] * PAGE for _ in range(p.num_pages)] for g, p in m.pools.items()}
        self.slots = [() for _ in range(m.slots.num_slots)]

    def step(self, rid, tokens):
        m = self.m
        at = m.length(rid)
        with m.lease([(rid, len(tokens))]):
            for g in self.pages:
                table = m.block_table(rid, g)
                for i, t in enumerate(tokens):
                    self.pages[g][table[(at + i) // PAGE]][(at + i) % PAGE] = t
            self.slots[m.slot(rid)] += tuple(tokens)

    def fork(self, copies):
        for g, pairs in copies.pages.items():
            for a, b in pairs:
                self.pages[g][b][: copies.tokens] = self.pages[g][a][: copies.tokens]
        for a, b in copies.slots:
            self.slots[b] = self.slots[a]

    def reorder(self, o):
        was = [self.slots[s] for s in o.slots]
        for s, p in zip(o.slots, o.parents):
            self.slots[s] = was[p]
        for g, rows in o.pages.items():
            was = [list(self.pages[g][p]) for p in rows]
            for page, p in zip(rows, o.parents):
                self.pages[g][page][: o.tokens] = was[p][: o.tokens]

    def compact(self, moves):
        for g, pairs in moves.items():
            for a, b in pairs:
                self.pages[g][b] = list(self.pages[g][a])

    def check(self, rid, tokens):
        m = self.m
        assert m.length(rid) == len(tokens) and self.slots[m.slot(rid)] == tuple(tokens)
        for g in self.pages:
            need, table = m.layout.groups[g].need, m.block_table(rid, g)
            for i in range(need.first_key_kept(len(tokens)), len(tokens)):
                assert self.pages[g][table[i // PAGE]][i % PAGE] == tokens[i], (rid, g, i)


@pytest.mark.parametrize("seed", range(12))
def test_families_keep_what_they_hold(seed):
    """Requests that step, fork, take over one another's state, close and move to other pages hold their own tokens throughout."""
    rng = random.Random(seed)
    m = manager(60, 12, *[(FULL, STATE), (FULL, WIN, STATE), (WIN, BLOCK), (STATE,)][seed % 4])
    dev, live, next_id = Device(m), {}, 0
    for _ in range(500):
        op, rid = rng.random(), rng.choice(list(live)) if live else None
        if op < 0.1 or rid is None:
            if len(live) < 12:
                dev.slots[m.open(next_id)] = ()
                live[next_id] = []
                next_id += 1
        elif op < 0.5:
            new = [rng.randrange(1000) for _ in range(rng.choice([1, 1, 2, 5]))]
            try:
                dev.step(rid, new)
                live[rid] = live[rid] + new
            except OutOfPages:
                pass
        elif op < 0.65:
            ids = [next_id + i for i in range(rng.randint(1, 3))]
            before = (m.free_pages(), m.slots.free_count)
            try:
                dev.fork(m.fork(rid, ids))
                live.update({i: list(live[rid]) for i in ids})
                next_id += len(ids)
            except (OutOfPages, OutOfSlots):
                assert before == (m.free_pages(), m.slots.free_count)
        elif op < 0.85:
            family = [i for i in live if m._req[i].family == m._req[rid].family and len(live[i]) == len(live[rid])]
            rng.shuffle(family)
            parents = [rng.randrange(len(family)) for _ in family]
            dev.reorder(m.reorder(family, parents))
            new = [live[family[p]] for p in parents]
            live.update({i: list(t) for i, t in zip(family, new)})
        elif op < 0.9:
            dev.compact(m.compact())
            for g, p in m.pools.items():
                held = {x for r in m._req.values() for x in r.tables[g] if x >= 0}
                assert held == set(range(len(held)))
        else:
            m.close(rid)
            del live[rid]
        m.check_invariants()
        for i, tokens in live.items():
            dev.check(i, tokens)
        families = {}
        for i in live:
            families.setdefault(m._req[i].family, []).append(i)
        for ids in families.values():
            some = rng.sample(ids, rng.randint(1, len(ids)))
            n = m.common_length(some)
            assert all(live[i][:n] == live[some[0]][:n] for i in some) and n <= min(len(live[i]) for i in some)
        if len(live) > 1:
            a, b = rng.sample(list(live), 2)
            if m._req[a].family != m._req[b].family:
                assert m.common_length([a, b]) == 0
    for i in list(live):
        m.close(i)
    m.check_invariants()
    assert all(n == 60 for n in m.free_pages().values())


def test_a_fork_shares_the_prompts_pages():
    m = manager(10, 4, FULL)
    m.open("a")
    with m.lease([("a", 10)]):
        pass
    c = m.fork("a", ["b", "c"])
    assert c.tokens == 2 and c.pages == {0: [(2, 3), (2, 4)]} and c.slots == [(0, 1), (0, 2)]
    assert m.block_table("b", 0) == [0, 1, 3] and m.free_pages() == {0: 5} and m.common_length(["a", "b", "c"]) == 10
    o = m.reorder(["a", "b", "c"], [1, 1, 0])
    assert o.pages == {0: [2, 3, 4]} and o.slots == [0, 1, 2] and o.tokens == 2 and o.parents == [1, 1, 0]
    m.close("a")
    assert m.free_pages() == {0: 6}                        # its own page alone
    m.close("b"); m.close("c")
    assert m.free_pages() == {0: 10}


def test_what_forks_refuse():
    m = manager(4, 3, FULL)
    m.open("a")
    with m.lease([("a", 9)]):
        with pytest.raises(RuntimeError):
            m.fork("a", ["b"])
        with pytest.raises(RuntimeError):
            m.compact()
    with pytest.raises(KeyError):
        m.fork("a", ["a"])
    with pytest.raises(KeyError):
        m.fork("a", ["b", "b"])
    with pytest.raises(KeyError):
        m.fork("x", ["b"])
    with pytest.raises(OutOfPages):
        m.fork("a", ["b", "c"])
    with pytest.raises(OutOfSlots):
        m.fork("a", ["b", "c", "d"])
    m.check_invariants()
    m.fork("a", ["b"])
    m.open("z")
    for ids, parents in ((["a", "b"], [0]), (["a", "b"], [0, 2]), (["a", "z"], [0, 0]), (["a", "a"], [0, 0])):
        with pytest.raises(ValueError):
            m.reorder(ids, parents)
    m.check_invariants()


@pytest.mark.parametrize("seed", range(30))
def test_rows_for_the_chosen(seed):
    rng = random.Random(seed)
    beams = rng.randint(1, 9)
    chosen = [(-float(i), rng.randrange(beams), 100 + i) for i in range(rng.randint(0, beams))]
    parents, rows = take_rows(chosen, beams)
    assert sorted((s, parents[r], t) for r, (s, t) in enumerate(rows) if s > -np.inf) == sorted(chosen)
    used = {p for _s, p, _t in chosen}
    assert all(parents[p] == p for p in used)              # a source stays, so the moves do not meet
    assert all(parents[r] == r for r, (s, _t) in enumerate(rows) if s == -np.inf)


def reference_search(log_probs, p, eos, room, held=float):
    """Beam search by its definition: `log_probs(tokens)` of the next token, all beams anew every step; `held`: what a running sum is held in."""
    beams, ended = [([], 0.0)], []
    for _ in range(room):
        cands = [(s + lp, b, t) for b, (seq, s) in enumerate(beams) for t, lp in enumerate(log_probs(seq))]
        cands.sort(key=lambda c: (-c[0], c[1], c[2]))
        live = []
        for rank, (s, b, t) in enumerate(cands[: p.beams * (1 + len(eos))]):
            if s == -np.inf:
                break
            seq, s = beams[b][0] + [t], float(held(s))
            if t in eos:
                if rank < p.beams:
                    ended.append((s / len(seq) ** p.length_penalty, s, seq, "stop"))
            elif len(live) < p.beams:
                live.append((seq, s))
        ended.sort(key=lambda e: -e[0])
        del ended[p.beams:]
        if not live:
            break
        beams = live
        n = len(live[0][0])
        if n == room:
            for seq, s in live:
                ended.append((s / n ** p.length_penalty, s, seq, "length"))
            ended.sort(key=lambda e: -e[0])
            del ended[p.beams:]
        elif len(ended) >= p.beams and (p.early_stopping or ended[-1][0] >= max(s for _q, s in live) / n ** p.length_penalty):
            break
    return ended[: p.best]


@pytest.mark.parametrize("seed", range(40))
def test_a_search_by_its_definition(seed):
    """`_Search` fed with each step's best against the definition, for a language whose next token hangs on the last two."""
    rng = np.random.default_rng(seed)
    vocab = int(rng.integers(3, 9))
    table = np.log(rng.dirichlet(np.full(vocab, 0.6), size=(vocab + 1, vocab + 1)))
    table[rng.random(table.shape) < 0.2] = -np.inf         # forbidden words
    log_probs = lambda seq: table[seq[-2] if len(seq) > 1 else vocab, seq[-1] if seq else vocab]  # noqa: E731
    p = BeamParams(beams=int(rng.integers(1, 6)), length_penalty=float(rng.choice([0.0, 1.0, 1.7, -0.5])), early_stopping=bool(rng.random() < 0.4))
    p = BeamParams(**{**p.__dict__, "best": p.beams})
    eos, room = set(rng.choice(vocab, int(rng.integers(0, 3)), replace=False).tolist()), int(rng.integers(1, 9))
    s, over = _Search(list(range(p.beams)), room), False
    held = [[]]                                            # what the rows hold, as a device would
    while not over:
        scores = s.scores or [0.0]
        cands = sorted(((scores[r] + lp, r, t) for r, seq in enumerate(held) for t, lp in enumerate(log_probs(seq))), key=lambda c: (-c[0], c[1], c[2]))
        parents, over = s.advance(cands[: p.beams * (1 + len(eos))], p, eos)
        held = [held[parents[r]] + [s.tokens[r][-1]] for r in range(p.beams)]
        assert held == s.tokens
    want = reference_search(log_probs, p, eos, room)
    assert [(h.tokens, h.finish_reason) for h in s.ended] == [(e[2], e[3]) for e in want]
    assert [h.score for h in s.ended] == pytest.approx([e[0] for e in want]) and [h.log_prob for h in s.ended] == pytest.approx([e[1] for e in want])


def test_params_are_checked():
    for kw in (dict(beams=0), dict(beams=65), dict(best=0), dict(beams=2, best=3), dict(max_tokens=0), dict(length_penalty=float("nan"))):
        with pytest.raises(ValueError):
            BeamParams(**kw).validate()


def test_the_operators_refuse_what_is_not_on_the_device():
    import torch
    from rustinfer_b200.ops import kernels as K
    from rustinfer_b200.ops.library import KernelError
    f, i = torch.zeros((4, 50)), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: K.beam_select(f, f[0, :4], 2, f[:2, :3], i, i), lambda: K.reorder_rows(f, i, i, 2), lambda: K.copy_pages(f, i, i),
                 lambda: K.attention_decode_beams(f, f, f, f, i, i, 2, 1, 1, 16, 1.0, None, 1, 1)):
        with pytest.raises(KernelError):
            call()
