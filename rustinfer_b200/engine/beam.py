"""Beam search over the step function: the `beams` best continuations of every prompt, side by side.

A prompt is computed once and forked: its beams share its pages.  Every step runs all beams of all prompts as single tokens
(the attention reads the keys of a prompt once for its beams), one kernel chooses the best continuations over beams and
vocabulary, and a beam whose continuations did not make it takes over the pages, the partly filled page and the fixed state of
one that has several.  A beam that has a continuation keeps its row, so only what has to move is moved.

RustInfer samples one continuation a request (crates/infer-worker/src/application/sampler_stack.rs:242-351); names of the
options follow its sampling parameters where they mean the same (crates/infer-core/src/ports/sampler.rs:18-47).
"""
from __future__ import annotations

import math
from dataclasses import dataclass, field
from typing import Any, Dict, List, Optional, Sequence, Tuple

import torch

from ..ops import kernels as K
from .runner import ModelRunner, StepEntry


@dataclass(frozen=True)
class BeamParams:
    beams: int = 4                      # continuations kept beside one another
    best: int = 1                       # of them returned, best first
    max_tokens: int = 16
    length_penalty: float = 1.0         # a hypothesis counts as log-probability / tokens ** length_penalty
    early_stopping: bool = False        # True: a prompt is done when `beams` hypotheses have ended; else when no live beam, as long as it is, is worth more
    ignore_eos: bool = False

    def validate(self) -> None:
        if not 1 <= self.beams <= K.BEAMS_MAX:
            raise ValueError(f"beams must lie in 1 to {K.BEAMS_MAX}")
        if not 1 <= self.best <= self.beams:
            raise ValueError("best must lie in 1 to beams")
        if self.max_tokens < 1:
            raise ValueError("max_tokens must be at least 1")
        if not self.length_penalty == self.length_penalty or abs(self.length_penalty) == float("inf"):
            raise ValueError("length_penalty must be finite")
        if abs(self.length_penalty) * math.log(self.max_tokens) > 600.0:       # e ** 600: a factor e ** 109 inside what 64 bits hold
            raise ValueError(f"length_penalty {self.length_penalty}: {self.max_tokens} tokens ** length_penalty leaves the range of 64 bits")


@dataclass
class BeamHypothesis:
    tokens: List[int]
    log_prob: float                     # sum over its tokens
    score: float                        # log_prob / tokens ** length_penalty
    finish_reason: str                  # "stop" (a stop id, its last token) or "length"


def take_rows(chosen: Sequence[Tuple[float, int, int]], beams: int) -> Tuple[List[int], List[Tuple[float, int]]]:
    """Rows for the chosen continuations (score, parent row, token; best first, up to `beams`): parents[r], and (score, token) of every
    row.  A parent's first continuation keeps its row, the others take the rows nobody continues, in ascending order; a row
    for which nothing is left stays as it is with a score of -inf."""
    parents, rows = list(range(beams)), [(float("-inf"), 0)] * beams
    kept, others = set(), []
    for score, parent, token in chosen:
        if parent in kept:
            others.append((score, parent, token))
        else:
            kept.add(parent)
            rows[parent] = (score, token)
    free = (r for r in range(beams) if r not in kept)
    for score, parent, token in others:
        r = next(free)
        parents[r], rows[r] = parent, (score, token)
    return parents, rows


@dataclass
class _Search:
    """One prompt's search: its rows, what they hold, and what has ended."""
    ids: List[Any]
    room: int                           # tokens that may be made: max_tokens, or less where max_model_len ends before
    tokens: List[List[int]] = field(default_factory=list)
    scores: List[float] = field(default_factory=list)
    ended: List[BeamHypothesis] = field(default_factory=list)

    def end(self, tokens: List[int], log_prob: float, p: BeamParams, reason: str) -> None:
        self.ended.append(BeamHypothesis(tokens, log_prob, log_prob / len(tokens) ** p.length_penalty, reason))
        self.ended.sort(key=lambda h: -h.score)            # stable: of equals the one that ended first
        del self.ended[p.beams:]

    def advance(self, picks: Sequence[Tuple[float, int, int]], p: BeamParams, eos: Sequence[int]) -> Tuple[List[int], bool]:
        """Takes a step's choice (score, row of this search, token; best first): the rows' parents, and whether the search is over.
        A continuation that ends with a stop id is a hypothesis if it is among the `beams` best."""
        live: List[Tuple[float, int, int]] = []
        for rank, (score, row, token) in enumerate(picks):
            if score == float("-inf"):
                break
            if token in eos:
                if rank < p.beams:
                    self.end((self.tokens[row] if self.tokens else []) + [token], score, p, "stop")
            elif len(live) < p.beams:
                live.append((score, row, token))
        n = p.beams if self.tokens else 1                  # the first choice has one row, the prompt's
        if self.tokens:
            parents, rows = take_rows(live, p.beams)
        else:
            rows = [(s, t) for s, _r, t in live] + [(float("-inf"), 0)] * (p.beams - len(live))
            parents = [0] * p.beams
        before = self.tokens or [[]] * n
        self.tokens = [before[parents[r]] + [rows[r][1]] for r in range(p.beams)]
        self.scores = [s for s, _t in rows]
        made = len(self.tokens[0])
        best = max(self.scores)
        over = best == float("-inf")
        if made >= self.room and not over:
            for s, t in zip(self.scores, self.tokens):
                if s > float("-inf"):
                    self.end(t, s, p, "length")
            over = True
        if len(self.ended) >= p.beams and not over:
            # the usual rule: no live beam, counted by its length now, comes to more than the worst that has ended (with a length_penalty above 0 one
            # that grew longer still could)
            over = p.early_stopping or self.ended[-1].score >= best / made ** p.length_penalty
        return parents, over


class BeamSearch:
    """Runs searches on a runner nobody else steps meanwhile."""

    def __init__(self, runner: ModelRunner, params: BeamParams, eos: Sequence[int]):
        params.validate()
        self.r, self.p = runner, params
        self.eos = set() if params.ignore_eos else set(eos)
        self.picks = params.beams * (1 + len(self.eos))    # as many that go on as there are beams, whatever ends
        if params.beams > runner.max_batch_seqs:
            raise ValueError(f"{params.beams} beams exceed max_batch_seqs {runner.max_batch_seqs}")
        if self.picks > K.BEAM_PICKS_MAX:
            raise ValueError(f"{params.beams} beams with {len(self.eos)} stop ids need {self.picks} picks a step, {K.BEAM_PICKS_MAX} are built")
        self.steps = 0

    def _pages(self, prompt: int) -> int:
        """Pages of a group a search may come to hold: its prompt's, and what every beam fills of its own."""
        ps = self.r.page_size
        end = min(prompt + self.p.max_tokens, self.r.max_model_len)
        return -(-prompt // ps) + self.p.beams * (-(-end // ps) - prompt // ps)

    def _choose(self, logits: torch.Tensor, scores: Sequence[float], beams: int) -> List[List[Tuple[float, int, int]]]:
        rows = logits.shape[0]
        picks = min(self.picks, beams * logits.shape[1])
        dev = logits.device
        best = torch.empty((3, rows // beams, picks), dtype=torch.int32, device=dev)
        K.beam_select(logits, torch.tensor(scores, dtype=torch.float32).pin_memory().to(dev, non_blocking=True), beams,
                      best[0].view(torch.float32), best[1], best[2])
        host = best.cpu()
        return [[(s, r - g * beams, t) for s, r, t in zip(*cols)]
                for g, cols in enumerate(zip(host[0].view(torch.float32).tolist(), host[1].tolist(), host[2].tolist()))]

    def _prefill(self, ids: Sequence[Any], prompts: Sequence[Sequence[int]]) -> torch.Tensor:
        """The logits behind every prompt, [prompts, vocab]."""
        r = self.r
        rows: List[torch.Tensor] = []
        at, i = 0, 0                                       # the prompt under way, and how far it is
        while i < len(prompts):
            entries, budget = [], r.max_batch_tokens
            while i < len(prompts) and budget > 0:
                part = list(prompts[i][at: at + budget])
                last = at + len(part) == len(prompts[i])
                entries.append(StepEntry(ids[i], part, [len(part) - 1] if last else []))
                budget -= len(part)
                at = 0 if last else at + len(part)
                i += last
                if not last:
                    break
            got = r.step(entries)
            self.steps += 1
            if got is not None:
                rows.append(got)
        return torch.cat(rows) if len(rows) > 1 else rows[0]

    def run(self, prompts: Sequence[Sequence[int]]) -> List[List[BeamHypothesis]]:
        r, p = self.r, self.p
        free = min(r.cache.free_pages().values(), default=1 << 60)
        for q in prompts:
            if not len(q):
                raise ValueError("an empty prompt")
            if len(q) >= r.max_model_len:
                raise ValueError(f"a prompt of {len(q)} tokens leaves no room under max_model_len {r.max_model_len}")
            if self._pages(len(q)) > free:
                raise ValueError(f"{p.beams} beams behind a prompt of {len(q)} tokens may need {self._pages(len(q))} cache pages, {free} are free")
        out: List[List[BeamHypothesis]] = []
        while len(out) < len(prompts):                     # as many prompts side by side as rows and pages allow
            wave: List[Sequence[int]] = []
            pages = free
            for q in prompts[len(out): len(out) + r.max_batch_seqs // p.beams]:
                pages -= self._pages(len(q))
                if pages < 0:
                    break
                wave.append(q)
            out += self._wave(wave, len(out))
        return out

    def _wave(self, prompts: Sequence[Sequence[int]], first: int) -> List[List[BeamHypothesis]]:
        r, p = self.r, self.p
        searches = [_Search([("beam", first + i, b) for b in range(p.beams)], min(p.max_tokens, r.max_model_len - len(q)))
                    for i, q in enumerate(prompts)]
        opened: Dict[Any, None] = {}
        try:
            for s in searches:
                r.open(s.ids[0])
                opened[s.ids[0]] = None
            logits = self._prefill([s.ids[0] for s in searches], prompts)
            active = []
            for s, picks in zip(searches, self._choose(logits, [0.0] * len(searches), 1)):
                if s.advance(picks, p, self.eos)[1]:
                    r.close(s.ids[0])
                    del opened[s.ids[0]]
                    continue
                r.fork(s.ids[0], s.ids[1:])
                opened.update(dict.fromkeys(s.ids[1:]))
                active.append(s)
            while active:
                rows = [i for s in active for i in s.ids]
                logits = r.step([StepEntry(i, [t[-1]], [0]) for s in active for i, t in zip(s.ids, s.tokens)], borrow_logits=True, beams=p.beams)
                self.steps += 1
                chosen = self._choose(logits, [x for s in active for x in s.scores], p.beams)
                parents, still = [], []
                for j, (s, picks) in enumerate(zip(active, chosen)):
                    up, over = s.advance(picks, p, self.eos)
                    # what is over moves nothing any more
                    parents += [j * p.beams + (b if over else x) for b, x in enumerate(up)]
                    if not over:
                        still.append(s)
                r.reorder(rows, parents, p.beams)
                for s in active:
                    if s not in still:
                        for i in s.ids:
                            r.close(i)
                            del opened[i]
                active = still
        finally:
            for i in opened:
                r.close(i)
        return [s.ended[: p.best] for s in searches]
