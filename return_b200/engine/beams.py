"""Beam search over the engine's step function.

The reference samples one continuation a request.  Here a prompt's ``beams`` best continuations are carried on side by side: a beam is a
request of the cache manager, all beams of all prompts decode in one step (through the captured graphs), one kernel selects the best
continuations of every prompt over its beams and the vocabulary (``ops.beam_select``), and a beam that is carried on more than once is
forked: its full pages are shared, the rows of its partly filled last page and its per-request states are copied
(``ModelRunner.fork_requests``).  The beam carried on first keeps its pages and its slot.  Where the pages do not suffice for all prompts
that search at once, the last one gives back what it holds and starts again behind the others; one that does not fit alone raises
``KVCapacityError``.

A continuation that ends with ``eos_token_id`` leaves the beams with the score (sum of its log-probabilities) / length ** length_penalty
if it is among the ``beams`` best of its step; the search of a prompt ends when ``beams`` have left and none that goes on has a higher
score than the lowest of them, or at ``max_new_tokens``.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence

import torch

from ..cache.manager import KVCapacityError
from ..ext import ops
from .batch import StepEntry


@dataclass
class BeamResult:
    output_ids: List[int]
    score: float                      # what the results are ordered by
    logprob: float                    # the sum of the tokens' log-probabilities
    finish_reason: str                # "stop" | "length"

    def as_dict(self) -> dict:
        return {"output_ids": self.output_ids, "score": self.score, "logprob": self.logprob, "finish_reason": self.finish_reason}


class _Search:
    """One prompt's beams: ``names`` of their requests, tokens and sums of log-probabilities, in order; what has left."""

    def __init__(self, index: int, prompt: Sequence[int]):
        self.index, self.prompt = index, list(prompt)
        self.serial = 0
        self.begin()

    def begin(self) -> None:
        self.names: List[tuple] = []
        self.tokens: List[List[int]] = []
        self.scores: List[float] = []
        self.parents: List[int] = []             # which beam of the step before each one goes on from
        self.left: List[BeamResult] = []

    def name(self) -> tuple:
        self.serial += 1
        return ("beam", self.index, self.serial)


class BeamSearch:
    def __init__(self, runner, beams: int, max_new_tokens: int, length_penalty: float = 1.0, eos_token_id: Optional[int] = None):
        V = runner.vocab_size
        if not 1 <= beams <= min(ops.BEAM_MAX_BEAMS, runner.config.max_reside):
            raise ValueError(f"beams: 1 to {ops.BEAM_MAX_BEAMS}, and no more than max_reside={runner.config.max_reside}")
        if max_new_tokens < 1:
            raise ValueError("max_new_tokens must be at least 1")
        # the beams that go on, and as many that may end: one word ends a continuation, so each beam offers one of those at most
        self.keep = 2 * beams if eos_token_id is not None else beams
        if V < self.keep or not (eos_token_id is None or 0 <= eos_token_id < V):
            raise ValueError(f"a vocabulary of {V} for {beams} beams, eos_token_id={eos_token_id}")
        self.runner, self.beams, self.max_new, self.penalty, self.eos = runner, beams, max_new_tokens, length_penalty, eos_token_id
        self._put_off: List[_Search] = []        # those of the prompts at hand that found no pages beside the others

    # ------------------------------------------------------------------ all prompts
    def run(self, prompts: Sequence[Sequence[int]]) -> List[List[BeamResult]]:
        r = self.runner
        for p in prompts:
            if not p:
                raise ValueError("a prompt needs at least one token")
            if len(p) + self.max_new - 1 > r.max_positions:
                raise KVCapacityError(f"a prompt of {len(p)} tokens and {self.max_new} new ones exceed the engine's sequence limit {r.max_positions}")
        searches = [_Search(i, p) for i, p in enumerate(prompts)]
        at_once, waiting = r.config.max_reside // self.beams, list(searches)
        while waiting:                                        # as many prompts at a time as have slots for all their beams
            group, waiting = waiting[:at_once], waiting[at_once:]
            self._put_off = []
            try:
                with torch.cuda.device(r.env.device):
                    self._run_group(group)
            finally:
                for s in group:
                    self._give_back(s)
            if self._put_off:
                at_once = max(1, len(group) - len(self._put_off))
                waiting = self._put_off[::-1] + waiting
        return [sorted(s.left, key=lambda h: -h.score)[:self.beams] for s in searches]

    def _give_back(self, s: _Search) -> None:
        for name in s.names:
            self.runner.free_request(name)
        s.names = []

    def _put_off_last(self, live: List[_Search]) -> None:
        s = live.pop()
        self._give_back(s)
        s.begin()
        self._put_off.append(s)

    def _run_group(self, group: List[_Search]) -> None:
        live = list(group)
        logits = self._prompts(live)
        for s in live:
            s.tokens, s.scores = [[]], [0.0]
        while True:
            picked = self._select(live, logits, len(live[0].names))
            for s, candidates in zip(live, picked):
                self._advance(s, candidates)
            for s in live:                                    # a search that is over gives back what its beams hold
                if not s.tokens:
                    self._give_back(s)
            live = [s for s in live if s.tokens]
            if not live:
                return
            self._fork(live)
            logits = self.runner.step(self._next_tokens(live))

    # ------------------------------------------------------------------ the pieces of a step
    def _prompts(self, live: List[_Search]) -> torch.Tensor:
        """Runs the prompts, portions of several in one step; the logits behind each prompt's last token, [prompts, vocab].  Prompts that
        find no pages leave ``live``."""
        r = self.runner
        rows: Dict[int, torch.Tensor] = {}
        done = {s.index: 0 for s in live}
        for s in live:
            name = s.name()
            r.add_request(name)
            s.names = [name]
        while any(done[s.index] < len(s.prompt) for s in live):
            budget, entries, ends = r.config.prefill_chunk, [], []
            for s in list(live):
                at = done[s.index]
                n = min(budget, len(s.prompt) - at)
                if n <= 0:
                    continue
                last = at + n == len(s.prompt)
                try:
                    entries.append(r.reserve(s.names[0], s.prompt[at:at + n], [n - 1] if last else []))
                except KVCapacityError:
                    if s is live[0]:
                        raise
                    while s in live:                          # those behind it hold no pages yet
                        self._put_off_last(live)
                    break
                if last:
                    ends.append(s.index)
                done[s.index] += n
                budget -= n
            if not entries:
                continue
            logits = r.step(entries)
            for k, i in enumerate(ends):
                rows[i] = logits[k:k + 1].clone()             # a captured step's logits are the graph's own: the next one writes over them
        return torch.cat([rows[s.index] for s in live])

    def _next_tokens(self, live: List[_Search]) -> List[StepEntry]:
        """An entry for every beam's last token."""
        out: List[List[StepEntry]] = []
        for s in list(live):
            if s not in live:                                 # put off for one before it
                break
            entries: List[StepEntry] = []
            while len(entries) < len(s.names):
                name, tokens = s.names[len(entries)], s.tokens[len(entries)]
                try:
                    entries.append(StepEntry(name, tokens[-1:], [0], self.runner.manager.append(name, 1)))
                except KVCapacityError:
                    if len(live) == 1:
                        raise
                    self._put_off_last(live)
                    if s not in live:
                        break
            else:
                out.append(entries)
        return [e for entries in out for e in entries]

    def _select(self, live: List[_Search], logits: torch.Tensor, beams: int):
        """For each search its best continuations, best first: (score, beam, token)."""
        dev, n = logits.device, len(live)
        keep = min(self.keep, beams * logits.shape[1])
        scores = torch.tensor([x for s in live for x in s.scores], dtype=torch.float32).to(dev)
        best = torch.empty((n, keep), dtype=torch.float32, device=dev)
        places = torch.empty((2, n, keep), dtype=torch.int32, device=dev)
        ops.beam_select(logits, scores, beams, best, places[0], places[1])
        values, (parents, tokens) = best.tolist(), places.tolist()
        ops.check_status(dev)                                 # the step and the selection are done: a bounded wait that gave up raises here
        return [list(zip(*row)) for row in zip(values, parents, tokens)]

    def _advance(self, s: _Search, candidates) -> None:
        """The search's beams behind this step; no beams if it is over."""
        tokens, scores, parents = [], [], []
        for rank, (score, beam, token) in enumerate(candidates):
            if token == self.eos:
                if rank < self.beams and score != float("-inf"):
                    s.left.append(self._result(s.tokens[beam] + [token], score, "stop"))
            elif len(tokens) < self.beams:
                tokens.append(s.tokens[beam] + [token])
                scores.append(score)
                parents.append(beam)
        s.left = sorted(s.left, key=lambda h: -h.score)[:self.beams]
        over = len(tokens[0]) >= self.max_new
        if over:
            s.left += [self._result(t, x, "length") for t, x in zip(tokens, scores) if x != float("-inf")]
        elif len(s.left) == self.beams:
            over = scores[0] / len(tokens[0]) ** self.penalty <= s.left[-1].score
        s.tokens, s.scores, s.parents = ([], [], []) if over else (tokens, scores, parents)

    def _result(self, tokens: List[int], score: float, reason: str) -> BeamResult:
        return BeamResult(list(tokens), score / len(tokens) ** self.penalty, score, reason)

    def _fork(self, live: List[_Search]) -> None:
        """Requests for the new beams: one that is carried on first keeps its request, one that is not gives back what it holds, all
        others are copies."""
        names: List[List[tuple]] = []
        copies: List[List[tuple]] = []
        for s in live:
            names.append([])
            copies.append([])
            going = set()
            for p in s.parents:
                if p in going:
                    names[-1].append(s.name())
                    copies[-1].append((s.names[p], names[-1][-1]))
                else:
                    going.add(p)
                    names[-1].append(s.names[p])
            for p, name in enumerate(s.names):
                if p not in going:
                    self.runner.free_request(name)
            s.names = [name for p, name in enumerate(s.names) if p in going]
        while any(copies):
            try:
                self.runner.fork_requests([pair for pairs in copies for pair in pairs])
                break
            except KVCapacityError:                           # nothing was copied
                if len(live) == 1:
                    raise
                self._put_off_last(live)
                names.pop()
                copies.pop()
        for s, now in zip(live, names):
            s.names = now
