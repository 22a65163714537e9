"""Beam search through the engine: every family's models against searches that compute every beam's logits from its whole
sequence anew, forks and reorders against requests that were never forked, and the calls that are refused."""
import math

import numpy as np
import pytest
import torch

import dirurax_helpers
import dozotar_helpers
import fotulix_helpers
import helpers
import linedra_helpers
import pikalix_helpers
import sotazen_helpers
from helpers import random_ids
from rustinfer_b200.weights.random_init import write_random_model
from test_beam_host import reference_search

pytestmark = pytest.mark.gpu

FAMILIES = {"llama": (helpers, ["A", "B", "C", "D", "E", "F"]), "dirurax": (dirurax_helpers, None), "pikalix": (pikalix_helpers, None),
            "sotazen": (sotazen_helpers, None), "linedra": (linedra_helpers, None), "dozotar": (dozotar_helpers, None),
            "fotulix": (fotulix_helpers, None)}
MODELS = [(f, n) for f, (h, names) in FAMILIES.items() for n in (names or sorted(h.CONFIGS))]
SOME = [("llama", "A"), ("llama", "D"), ("llama", "E")] + [(f, sorted(h.CONFIGS)[0]) for f, (h, names) in FAMILIES.items() if names is None]


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    made = {}

    def get(family, name):
        if (family, name) not in made:
            h = FAMILIES[family][0]
            cfg = h.TINY[name] if family == "llama" else h.config_json(name) if hasattr(h, "config_json") else h.CONFIGS[name]
            # weights that leave the next token open: continuations of a sharp model tie
            made[family, name] = write_random_model(str(tmp_path_factory.mktemp(f"{family}_{name}")), cfg, seed=5, std=0.12, norm_std=0.1)
        return made[family, name]
    return get


def _engine(folder, dtype, **kw):
    from rustinfer_b200.engine.engine import Engine
    args = dict(max_batch_seqs=12, max_model_len=128, paged_block_size=8, num_blocks=200, max_batch_tokens=128, capture_sizes=[])
    args.update(kw)
    eng = Engine(folder, dtype=dtype, **args)
    eng.runner.beam_keys = 0                               # however few keys they share, beams read them together
    return eng


def _log_probs(runner, prompt):
    """log-probabilities of the token behind prompt + seq, from a request of its own."""
    from rustinfer_b200.engine.runner import StepEntry

    def of(seq):
        runner.open("anew")
        ids = list(prompt) + list(seq)
        for at in range(0, len(ids), runner.max_batch_tokens):
            part = ids[at: at + runner.max_batch_tokens]
            x = runner.step([StepEntry("anew", part, [len(part) - 1])])
        runner.close("anew")
        return torch.log_softmax(x[0].double(), -1).tolist()
    return of


def _same(got, want):
    assert [(h.tokens, h.finish_reason) for h in got] == [(e[2], e[3]) for e in want]
    for h, e in zip(got, want):                            # a running sum in 32 bits, rounded once a token: 2^-24 of what it comes to
        bound = (len(h.tokens) + 1) * (2.0 ** -24 * abs(e[1]) + 2 * 2.0 ** -24 * 58 + 2.0 ** -22)
        assert abs(h.log_prob - e[1]) <= bound and abs(h.score - e[0]) <= bound


@pytest.mark.parametrize("family,name", MODELS)
def test_searches_in_32_bits(folder, family, name):
    """The 32-bit engine's logits do not depend on how a sequence was cut, so the search and one that computes every beam anew
    choose alike; prompts that end inside a page and at its end, several in a step."""
    from rustinfer_b200.engine.beam import BeamParams
    eng = _engine(folder(family, name), "float32")
    vocab = eng.runner.spec.vocab_size
    prompts = [random_ids(n, vocab, n + 3) for n in (5, 16, 1)]
    p = BeamParams(beams=3, best=3, max_tokens=12, ignore_eos=True)
    got = eng.beam_search(prompts, p)
    for prompt, hyps in zip(prompts, got):
        _same(hyps, reference_search(_log_probs(eng.runner, prompt), p, set(), 12, np.float32))
    eng.runner.cache.check_invariants()
    assert not eng.runner.cache.live_requests()


@pytest.mark.parametrize("beams,early,penalty", [(1, False, 1.0), (2, True, 1.0), (5, False, 0.0), (4, False, 2.0)])
def test_searches_that_end(folder, beams, early, penalty):
    """Stop ids, prompts in several waves, a search that ends while others go on."""
    from rustinfer_b200.engine.beam import BeamParams, BeamSearch
    eng = _engine(folder("llama", "A"), "float32", max_batch_tokens=40)
    vocab = eng.runner.spec.vocab_size
    prompts = [random_ids(n, vocab, n) for n in (3, 60, 8, 9, 30, 2)]
    eos = set(range(0, vocab, 9))
    while len(eos) > 128 // beams - 1:
        eos.pop()
    p = BeamParams(beams=beams, best=beams, max_tokens=9, length_penalty=penalty, early_stopping=early)
    got = BeamSearch(eng.runner, p, sorted(eos)).run(prompts)
    for prompt, hyps in zip(prompts, got):
        _same(hyps, reference_search(_log_probs(eng.runner, prompt), p, eos, 9, np.float32))
    if penalty <= 1:                                       # (a penalty of 2 leaves the longest alone)
        assert any(h.finish_reason == "stop" for hyps in got for h in hyps)
    assert not eng.runner.cache.live_requests()


@pytest.mark.parametrize("family,name", SOME)
def test_searches_from_captured_steps(folder, family, name):
    """Captured steps choose what eager ones choose, call after call.  (In 32 bits: the chained products of the bfloat16 engine add
    their slices in no fixed order.)"""
    from rustinfer_b200.engine.beam import BeamParams
    dtype = "float32"
    path = folder(family, name)
    eager, graph = _engine(path, dtype), _engine(path, dtype, capture_sizes=[1, 2, 4, 8])
    prompts = [random_ids(n, eager.runner.spec.vocab_size, n) for n in (20, 33)]
    for beams in (4, 3):
        p = BeamParams(beams=beams, best=beams, max_tokens=20, ignore_eos=True)
        a, b = eager.beam_search(prompts, p), graph.beam_search(prompts, p)
        assert [[(h.tokens, h.log_prob) for h in x] for x in a] == [[(h.tokens, h.log_prob) for h in x] for x in b]
    assert graph.runner.graph_replays > 30 and eager.runner.graph_replays == 0


@pytest.mark.parametrize("family,name", [m for m in SOME if m[0] == "llama"])
@pytest.mark.parametrize("sizes,beams", [([], 4), ([4, 8], 4), ([4, 8], 3)])
def test_what_a_hypothesis_is_worth_in_16_bits(folder, family, name, sizes, beams):
    """The log-probability a search reports against the one that its tokens get, read as a prompt: two ways through bfloat16
    kernels, so each token's may differ by what the logits do (the bound the ways of decoding are held to elsewhere: 6e-2 of
    the largest logit)."""
    from rustinfer_b200.engine.beam import BeamParams
    from rustinfer_b200.engine.runner import StepEntry
    eng = _engine(folder(family, name), "bfloat16", max_model_len=256, paged_block_size=16, capture_sizes=sizes)
    r = eng.runner
    prompts = [random_ids(n, r.spec.vocab_size, n) for n in (50, 100)]
    for prompt, hyps in zip(prompts, eng.beam_search(prompts, BeamParams(beams=beams, best=beams, max_tokens=15, ignore_eos=True))):
        for h in hyps:
            r.open("read")
            ids = prompt + h.tokens[:-1]
            x = r.step([StepEntry("read", ids, list(range(len(prompt) - 1, len(ids))))])
            r.close("read")
            lp = torch.log_softmax(x.double(), -1).gather(1, torch.tensor(h.tokens, device="cuda")[:, None]).sum()
            assert abs(float(lp) - h.log_prob) <= len(h.tokens) * 2 * 6e-2 * float(x.abs().max())


@pytest.mark.parametrize("family,name", SOME)
@pytest.mark.parametrize("sizes", [[], [4]])
def test_forks_and_reorders_of_requests(folder, family, name, sizes):
    """Forked, stepped apart, taken over from one another in a cycle, moved to other pages: every request's logits are those of
    one that was never forked."""
    from rustinfer_b200.engine.runner import ModelRunner, StepEntry
    r = ModelRunner(folder(family, name), dtype="float32", max_model_len=128, page_size=8, num_pages=80, max_batch_seqs=6, max_batch_tokens=128,
                    capture_sizes=sizes)
    r.beam_keys = 0
    vocab = r.spec.vocab_size
    held = {"a": random_ids(21, vocab, 1)}
    r.open("z")                                            # a neighbour, so that pages and slots lie apart
    r.step([StepEntry("z", random_ids(30, vocab, 2), [0])])
    r.open("a")
    r.step([StepEntry("a", held["a"], [0])])
    r.fork("a", ["b", "c", "d"])
    r.fork("a", [])
    held.update({i: list(held["a"]) for i in "bcd"})
    order, step = list("abcd"), 0

    def check():
        nonlocal step
        step += 1
        new = random_ids(4, vocab, 100 + step)
        x = r.step([StepEntry(i, [t], [0]) for i, t in zip(order, new)], beams=4)
        for i, t in zip(order, new):
            held[i].append(t)
        for k, i in enumerate(order):
            r.open("anew")
            want = r.step([StepEntry("anew", held[i], [len(held[i]) - 1])])
            r.close("anew")
            # (the bits of the Llama models do not hang on the cut; some recurrences' and experts' sums do, by a few 2^-24 a sum)
            near = 0.0 if family == "llama" else 2e-5 * float(want.abs().max())
            assert float((x[k] - want[0]).abs().max()) <= near, (i, step)

    for n in range(9):
        check()
        if n == 1:
            r.reorder(order, [1, 2, 3, 0])
            held = {i: list(held[order[p]]) for i, p in zip(order, [1, 2, 3, 0])}
        elif n == 3:
            r.reorder(order, [0, 0, 3, 3], beams=2)
            held = {i: list(held[order[p]]) for i, p in zip(order, [0, 0, 3, 3])}
        elif n == 4:
            r.close("z")
            assert r.compact() > 0 and r.compact() == 0
        elif n == 6:
            r.reorder(order, [2, 2, 2, 1])
            held = {i: list(held[order[p]]) for i, p in zip(order, [2, 2, 2, 1])}
    r.cache.check_invariants()
    for i in order:
        r.close(i)
    assert r.cache.free_pages() == {g: 80 for g in r.layout.paged_groups()}


def test_few_common_keys_are_read_row_by_row(folder):
    """Below `beam_keys` a step of beams is a step of rows; from there on one of beams."""
    from rustinfer_b200.engine.beam import BeamParams
    eng = _engine(folder("llama", "D"), "bfloat16", capture_sizes=[4])
    r, prompt = eng.runner, random_ids(40, 1000, 3)
    for keys, graphs in ((4 * 40 + 1, [4]), (4 * 40, [4, (4, 4)])):
        r.beam_keys = keys
        eng.beam_search([prompt], BeamParams(beams=4, max_tokens=4, ignore_eos=True))
        assert sorted(r._graphs, key=str) == sorted(graphs, key=str)


def test_requests_that_follow_a_search(folder):
    """The scheduler's requests get what they get on an engine that never searched.  (In 32 bits: the bfloat16 engine's own tokens differ
    now and then from run to run, without any search too, since its chained products add their slices in no fixed order.)"""
    from rustinfer_b200.engine.beam import BeamParams
    from rustinfer_b200.sampling.params import SamplingParams
    path = folder("llama", "D")
    a, b = (_engine(path, "float32", capture_sizes=[1, 2, 4]) for _ in range(2))
    prompts = [random_ids(n, a.runner.spec.vocab_size, n) for n in (9, 40, 17)]
    a.beam_search(prompts, BeamParams(beams=4, max_tokens=8, ignore_eos=True))
    a.beam_search(prompts[:1], BeamParams(beams=6, max_tokens=8, ignore_eos=True))
    sp = SamplingParams(max_tokens=12, ignore_eos=True)
    assert [x.tokens for x in a.generate(prompts, sp)] == [x.tokens for x in b.generate(prompts, sp)]


def test_what_a_search_refuses(folder):
    from rustinfer_b200.engine.beam import BeamParams
    from rustinfer_b200.engine.runner import StepEntry, StepError
    eng = _engine(folder("llama", "A"), "float32", num_blocks=20)
    r = eng.runner
    for prompts, p in (([[]], BeamParams()), ([[1] * 128], BeamParams()), ([[1] * 60], BeamParams(beams=8, max_tokens=60)),
                       ([[1]], BeamParams(beams=13)), ([[1]], BeamParams(beams=0)), ([[1]], BeamParams(best=5))):
        with pytest.raises(ValueError):
            eng.beam_search(prompts, p)
    assert eng.beam_search([], BeamParams()) == []
    with pytest.raises(StepError):
        eng.beam_search([[99999]], BeamParams())
    assert not r.cache.live_requests() and r.cache.free_pages() == {0: 20}
    r.open("a")
    r.step([StepEntry("a", [1, 2, 3], [0])])
    r.fork("a", ["b", "c"])
    with pytest.raises(StepError):
        r.step([StepEntry(i, [1], [0]) for i in "abc"], beams=2)
    with pytest.raises(StepError):
        r.step([StepEntry("a", [1, 2], [0]), StepEntry("b", [1, 2], [0])], beams=2)
    for parents, k in (([0, 1], None), ([0, 1, 3], None), ([1, 0, 0], 2), ([0, 0, 1], 65)):
        with pytest.raises(ValueError):
            r.reorder(list("abc"), parents, k)
    for i in "abc":
        r.close(i)
    eng.add_request([1, 2, 3])
    with pytest.raises(RuntimeError):
        eng.beam_search([[1]], BeamParams())


def test_a_prompt_that_leaves_room_for_little(folder):
    """max_model_len ends the hypotheses."""
    from rustinfer_b200.engine.beam import BeamParams
    eng = _engine(folder("llama", "A"), "float32", max_model_len=32)
    prompt = random_ids(29, eng.runner.spec.vocab_size, 7)
    p = BeamParams(beams=3, best=3, max_tokens=10, ignore_eos=True)
    (hyps,) = eng.beam_search([prompt], p)
    _same(hyps, reference_search(_log_probs(eng.runner, prompt), p, set(), 3, np.float32))
    assert all(len(h.tokens) == 3 and h.finish_reason == "length" and math.isfinite(h.score) for h in hyps)


def test_the_command_line_searches(folder, tmp_path, capsys):
    import json
    from rustinfer_b200 import cli
    from rustinfer_b200.engine.beam import BeamParams
    path = folder("llama", "A")
    run = tmp_path / "run.toml"
    run.write_text(f'model = "{path}"\ndtype = "float32"\nmax_model_len = 64\nnum_blocks = 40\nmax_batch_seqs = 4\ncapture_sizes = []\n'
                   '[sampling]\nbeams = 3\nbest = 2\nmax_tokens = 5\nignore_eos = true\n[[request]]\nprompt_ids = [5, 17, 3]\n')
    assert cli.main(["--config", str(run)]) == 0
    lines = [json.loads(l) for l in capsys.readouterr().out.splitlines()]
    want = _engine(path, "float32").beam_search([[5, 17, 3]], BeamParams(beams=3, best=2, max_tokens=5, ignore_eos=True))[0]
    assert [l["tokens"] for l in lines] == [h.tokens for h in want] and len(lines) == 2
