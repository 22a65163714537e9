"""Steps of beams of the bfloat16 engine, eager and captured: what every layer's attention is given (tables, lengths, common keys) and what
it returns, behind forks, reorders, a compaction and padding rows, against 64 bits over the keys and values that the requests have made."""
import pytest
import torch

import helpers
from helpers import random_ids
from rustinfer_b200.weights.random_init import write_random_model
from test_gpu_beams import _near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    made = {}

    def get(name):
        if name not in made:
            made[name] = write_random_model(str(tmp_path_factory.mktemp(name)), helpers.TINY[name], seed=5, std=0.12, norm_std=0.1)
        return made[name]
    return get


@pytest.fixture
def calls(monkeypatch):
    """Every call of the attention of beams; what it was given and returned, copied behind it (in a captured step by the step itself)."""
    from rustinfer_b200.ops import kernels
    real, seen = kernels.attention_decode_beams, []

    def spy(q, out, cache, block_table, kv_len, shared_len, *args):
        real(q, out, cache, block_table, kv_len, shared_len, *args)
        seen.append([t.clone() for t in (q, out, block_table, kv_len, shared_len)] + [cache, args])
    monkeypatch.setattr(kernels, "attention_decode_beams", spy)
    return seen


def _runner(path, **kw):
    from rustinfer_b200.engine.runner import ModelRunner
    args = dict(dtype="bfloat16", max_model_len=256, page_size=16, num_pages=90, max_batch_seqs=10, max_batch_tokens=256, capture_sizes=[])
    args.update(kw)
    r = ModelRunner(path, **args)
    r.beam_keys = 0                                        # however few keys they share, beams read them together
    return r


class Held:
    """Keys and values of every layer that each request has made or taken over, by position."""

    def __init__(self, r):
        self.r, self.kv = r, {}
        self.layers, self.page = r.group_storage[0], r.page_size

    def add(self, rid, upto):
        """The positions that are not held yet, from where the request's table says."""
        first = self.kv[rid].shape[1] if rid in self.kv else 0
        at = torch.arange(first, upto, device="cuda")
        table = torch.tensor(self.r.cache.block_table(rid, 0), device="cuda")
        new = self.layers[:, table[at // self.page], :, :, at % self.page]         # [positions, layers, K|V, kv heads, dim]
        new = new.transpose(0, 1).clone()
        self.kv[rid] = torch.cat([self.kv[rid], new], 1) if rid in self.kv else new


def _step_and_check(r, held, calls, saved, order, beams, seed, common):
    from rustinfer_b200.engine.runner import StepEntry
    new = random_ids(len(order), r.spec.vocab_size, seed)
    x = r.step([StepEntry(i, [t], [0]) for i, t in zip(order, new)], beams=beams)
    assert bool(x.isfinite().all())
    lengths = [r.cache.length(i) for i in order]
    for i, n in zip(order, lengths):
        held.add(i, n)
    if calls:                                              # an eager step, or the capture of one
        layers = held.layers.shape[0]
        assert len(calls) % layers == 0
        saved[:] = calls[-layers:]
        calls.clear()
    for layer, (q, out, table, kv_len, shared, cache, args) in enumerate(saved):
        of_beams, heads, kv_heads, dim, scale, window = args[:6]
        assert cache.data_ptr() == held.layers[layer].data_ptr() and of_beams == beams and window is None
        assert kv_len[: len(order)].tolist() == lengths and shared[: len(common)].tolist() == common
        assert all(int(n) == 1 for n in kv_len[len(order):]) and all(int(s) == 0 for s in shared[len(common):])
        for k, i in enumerate(order):
            want = r.cache.block_table(i, 0)
            assert table[k, : len(want)].tolist() == want, (i, layer)
            kv = held.kv[i][layer].double()
            p = torch.softmax(torch.einsum("kgd,tkd->kgt", q[k].double().view(kv_heads, heads // kv_heads, dim), kv[:, 0]) * scale, -1)
            got = torch.einsum("kgt,tkd->kgd", p, kv[:, 1]).reshape(1, -1)
            _near(out[k: k + 1], got, torch.einsum("kgt,tkd->kgd", p, kv[:, 1].abs()).reshape(1, -1), dim, len(kv))


@pytest.mark.parametrize("name,page", [("A", 16), ("D", 16), ("D", 8), ("E", 16)])
@pytest.mark.parametrize("sizes", [[], [8]])
def test_what_steps_of_beams_read(folder, calls, name, page, sizes):
    from rustinfer_b200.engine.runner import StepEntry
    r = _runner(folder(name), page_size=page, num_pages=1200 // page, capture_sizes=sizes)
    vocab, held, saved, beams = r.spec.vocab_size, Held(r), [], 3
    prompts = {"a": random_ids(50, vocab, 1), "b": random_ids(96, vocab, 2)}        # one ends inside a page, one at its end
    r.open("z")                                            # a neighbour, so that pages lie apart
    r.step([StepEntry("z", random_ids(30, vocab, 3), [0])])
    for f, prompt in prompts.items():
        r.open(f + "0")
        r.step([StepEntry(f + "0", prompt, [0])])
        r.fork(f + "0", [f + "1", f + "2"])
        held.add(f + "0", len(prompt))
        held.kv.update({f + k: held.kv[f + "0"] for k in "12"})
    order, common = [f + k for f in "ab" for k in "012"], [50, 96]
    moves = {1: [1, 2, 0, 5, 5, 5], 4: [0, 0, 1, 3, 4, 4], 7: [2, 2, 2, 4, 5, 3], 12: [1, 0, 2, 4, 4, 4], 17: [2, 1, 0, 3, 3, 5]}
    for n in range(22):                                    # (past two pages of 8 tokens and one of 16)
        _step_and_check(r, held, calls, saved, order, beams, 100 + n, common)
        if n in moves:
            r.reorder(order, moves[n], beams)
            held.kv = {i: held.kv[order[p]] for i, p in zip(order, moves[n])}
        elif n == 9:
            r.close("z")
            assert r.compact() > 0
    r.cache.check_invariants()
    assert (r.graph_replays > 0) == bool(sizes) and sorted(r._graphs) == ([(9, 3)] if sizes else [])
    # the rows of another family in the same places: nothing of the tables before is left
    for i in order[:3]:
        r.close(i)
    r.open("c0")
    r.step([StepEntry("c0", random_ids(61, vocab, 4), [0])])
    r.fork("c0", ["c1", "c2"])
    held.kv = {i: held.kv[i] for i in order[3:]}
    held.add("c0", 61)
    held.kv.update({"c1": held.kv["c0"], "c2": held.kv["c0"]})
    order, common = order[3:] + ["c0", "c1", "c2"], [96, 61]
    for n in range(3):
        _step_and_check(r, held, calls, saved, order, beams, 200 + n, common)
    _step_and_check(r, held, calls, saved, order[3:], beams, 300, [61])     # fewer rows of the same captured step
    _step_and_check(r, held, calls, saved, order, beams, 301, [96, 61])
    r.check_kernel_errors()


def test_requests_of_several_families_share_nothing(folder, calls):
    """A step that says that strangers are beams of one request: every row reads its own keys."""
    from rustinfer_b200.engine.runner import StepEntry
    r = _runner(folder("D"))
    held, saved = Held(r), []
    for i, n in (("a", 40), ("b", 40), ("c", 7), ("d", 100)):
        r.open(i)
        r.step([StepEntry(i, random_ids(n, r.spec.vocab_size, n), [0])])
        held.add(i, n)
    _step_and_check(r, held, calls, saved, ["a", "b", "c", "d"], 2, 5, [0, 0])
    _step_and_check(r, held, calls, saved, ["a", "b", "c", "d"], 4, 6, [0])


@pytest.mark.parametrize("sizes", [[], [66]])
def test_more_beams_than_are_read_together(folder, calls, sizes):
    """More than 64 forks of one request in a step are read row by row; the logits are those of steps of 33 and 33, to the bound that the ways
    of decoding are held to elsewhere (6e-2 of the largest logit)."""
    from rustinfer_b200.engine.runner import StepEntry
    r = _runner(folder("D"), max_batch_seqs=140, num_pages=400, capture_sizes=sizes)
    prompt = random_ids(40, r.spec.vocab_size, 1)
    r.open(0)
    r.step([StepEntry(0, prompt, [0])])
    r.fork(0, list(range(1, 132)))
    new = random_ids(66, r.spec.vocab_size, 2)
    x = r.step([StepEntry(i, [t], [0]) for i, t in enumerate(new)], beams=66).clone()
    assert not calls
    y = r.step([StepEntry(66 + i, [t], [0]) for i, t in enumerate(new)], beams=33)
    assert calls
    assert float((x - y).abs().max()) <= 6e-2 * float(y.abs().max())


def test_steps_take_the_sooner_way(tmp_path):
    """Without a number in `beam_keys` a step reads together while that is the sooner way: behind enough common keys, until there are too many own
    ones, from a captured step of its own kind; the 32-bit engine and few rows never."""
    from rustinfer_b200.engine.runner import StepEntry
    cfg = dict(helpers.TINY["E"], num_attention_heads=8, num_key_value_heads=8, max_position_embeddings=9000)
    path = write_random_model(str(tmp_path), cfg, seed=5, std=0.12, norm_std=0.1)
    for dtype, families, common, together in (("bfloat16", "ab", 8100, True), ("bfloat16", "ab", 7000, False), ("bfloat16", "a", 8100, False),
                                              ("float32", "ab", 8100, False)):
        r = _runner(path, dtype=dtype, max_model_len=9000, num_pages=1300, max_batch_tokens=64, capture_sizes=[8])
        r.beam_keys = None
        ids = [f + k for f in families for k in "0123"]
        for f in families:
            r.open(f + "0")
            with r.cache.lease([(f + "0", common)]):       # keys of zeros: what they are does not matter
                pass
            r.fork(f + "0", [f + k for k in "123"])
        for own, chosen in ((0, together), (60, together), (500, False)):
            for i in ids:
                with r.cache.lease([(i, common + own - r.cache.length(i))]):
                    pass
            r._graphs.clear()
            x = r.step([StepEntry(i, [5], [0]) for i in ids], beams=4)
            assert bool(x.isfinite().all()) and list(r._graphs) == [(8, 4) if chosen else 8], (dtype, families, common, own)


@pytest.mark.parametrize("name", ["A", "D", "E"])
def test_captured_steps_by_their_own_keys(folder, calls, name):
    """Beams with more than 96 keys of their own run from a captured step that is cut for more; both read what they should."""
    from rustinfer_b200.engine.runner import StepEntry
    r = _runner(folder(name), max_model_len=512, num_pages=150, capture_sizes=[6])
    vocab, held, order = r.spec.vocab_size, Held(r), [f + k for f in "ab" for k in "012"]
    saved, common = {}, [50, 96]
    for f, n in zip("ab", common):
        r.open(f + "0")
        r.step([StepEntry(f + "0", random_ids(n, vocab, n), [0])])
        r.fork(f + "0", [f + "1", f + "2"])
        held.add(f + "0", n)
        held.kv.update({f + k: held.kv[f + "0"] for k in "12"})
    for at, (own, key) in enumerate(((0, (6, 3)), (95, (6, 3)), (96, (6, 3, 200)), (230, (6, 3, 200)))):
        for i in order:
            more = own + common["ab".index(i[0])] - r.cache.length(i)
            if more > 0:
                r.step([StepEntry(i, random_ids(more, vocab, 7 * at + order.index(i)), [])])
                held.add(i, r.cache.length(i))
        _step_and_check(r, held, calls, saved.setdefault(key, []), order, 3, 50 + at, common)
        assert key in r._graphs and len(r._graphs) == 1 + (own >= 96)
        r.reorder(order, [1, 1, 0, 3, 5, 4], 3)
        held.kv = {i: held.kv[order[p]] for i, p in zip(order, [1, 1, 0, 3, 5, 4])}
