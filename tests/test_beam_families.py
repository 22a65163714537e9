"""Reorders of several families at once, on the host: all of them or none."""
import copy

import pytest

from rustinfer_b200.parts.base import FixedState, PagedKV
from test_beam_host import Device, manager

FULL, STATE = PagedKV(2, 16, None), FixedState((8,), "float32")


def _two_families():
    """a0 .. a2 and b0 .. b2, forked at 6 tokens and 3 more each on pages of 4."""
    m = manager(60, 8, FULL, STATE)
    dev, held = Device(m), {}
    for f, at in (("a", 0), ("b", 500)):
        dev.slots[m.open(f + "0")] = ()
        held[f + "0"] = list(range(at, at + 6))
        dev.step(f + "0", held[f + "0"])
        dev.fork(m.fork(f + "0", [f + "1", f + "2"]))
        for i in range(3):
            new = [at + 100 * (i + 1) + k for k in range(3)]
            held[f"{f}{i}"] = list(range(at, at + 6)) + new
            dev.step(f"{f}{i}", new)
    return m, dev, held


def _state(m):
    return copy.deepcopy((m._req, {g: p._holders for g, p in m.pools.items()}, {g: sorted(p._free) for g, p in m.pools.items()}))


IDS = ["a0", "a1", "a2", "b0", "b1", "b2"]


def test_families_are_taken_over_together():
    m, dev, held = _two_families()
    parents = [1, 2, 0, 5, 5, 5]
    for o in m.reorder_families(IDS, parents, 3):
        dev.reorder(o)
    m.check_invariants()
    for i, p in zip(IDS, parents):
        dev.check(i, held[IDS[p]])


@pytest.mark.parametrize("what", ["lengths", "another family", "not open", "twice", "parent of another family", "parents", "beams", "lease"])
def test_a_family_that_is_refused_leaves_the_others_as_they_were(what):
    m, dev, held = _two_families()
    ids, parents, beams, error, lease = list(IDS), [1, 2, 0, 4, 5, 3], 3, ValueError, None
    if what == "lengths":
        dev.step("b2", [7])
        held["b2"] = held["b2"] + [7]
    elif what == "another family":
        dev.slots[m.open("c")] = ()
        dev.step("c", list(range(9)))
        held["c"] = list(range(9))
        ids[5] = "c"
    elif what == "not open":
        ids[4], error = "x", KeyError
    elif what == "twice":
        ids[3:] = ids[:3]
    elif what == "parent of another family":
        parents[5] = 2
    elif what == "parents":
        parents = parents[:5]
    elif what == "beams":
        beams = 4
    else:
        lease, error = m.lease([("b0", 1)]), RuntimeError
    was = _state(m)
    with pytest.raises(error):
        m.reorder_families(ids, parents, beams)
    assert _state(m) == was
    if lease:
        lease.release()
    m.check_invariants()
    for i, tokens in held.items():
        dev.check(i, tokens)
