"""Beam search and scoring over the step function: continuations of one prompt that share its pages.

A beam is a request of the cache.  The prompt runs once; its beams are continuations of it (:meth:`CacheManager.fork`), which
hold its full pages together, and a decode step reads those once for all beams of a prompt where that pays (``plan.sharing_pays``).
Every step asks each beam's logits for its most probable tokens and their log probabilities (``kernels.token_logprobs``); the best
``width`` of all beams' go on: a beam chosen more than once is forked, one chosen no more is let go, all copies of a step in one
launch.  Not in the reference, whose server takes one sequence a request (src/engine/types.rs:14-37).
"""

from __future__ import annotations

import math
from dataclasses import dataclass, field
from typing import Dict, FrozenSet, Hashable, List, Optional, Sequence, Tuple

import torch

from .. import kernels
from ..sampling.sampler import InvalidLogits
from .scheduler import FINISH_LENGTH, FINISH_STOP, RequestRejected
from .step import StepEntry, StepError, Stepper


@dataclass
class BeamOutput:
    """One continuation: its tokens, their log probabilities, and the score that it was ranked by."""

    token_ids: List[int]
    token_logprobs: List[float]
    score: float
    finish_reason: str

    @property
    def logprob(self) -> float:
        return math.fsum(self.token_logprobs)


@dataclass
class TokenScores:
    """What a model makes of a sequence: for every token but the first its log probability given those in front of it, the
    entropy of what the model expected there, and (``alternatives`` > 0) the tokens that it held most probable, best first."""

    token_ids: List[int]
    logprobs: List[float]
    entropies: List[float]
    alternatives: List[List[Tuple[int, float]]] = field(default_factory=list)

    @property
    def logprob(self) -> float:
        return math.fsum(self.logprobs)

    @property
    def perplexity(self) -> float:
        return math.exp(-self.logprob / len(self.logprobs)) if self.logprobs else 1.0


@dataclass
class _Beam:
    request: Hashable
    tokens: List[int]
    logprobs: List[float]
    total: float


@dataclass
class _Search:
    """The beams of one prompt."""

    index: int
    prompt: List[int]
    beams: List[_Beam]
    finished: List[BeamOutput] = field(default_factory=list)


def _rank(total: float, length: int, penalty: float) -> float:
    return total / (max(1, length) ** penalty)


class BeamSearch:
    """``width`` beams a prompt, up to ``max_tokens`` tokens each.  A sequence's score is the sum of its tokens' log probabilities,
    divided by their number to the power of ``length_penalty``.  A beam that would go on with one of ``end_ids`` is finished there;
    a prompt is done when ``width`` of its continuations are finished or the beams have ``max_tokens`` tokens."""

    def __init__(self, stepper: Stepper, width: int, max_tokens: int, *, end_ids: FrozenSet[int] = frozenset(),
                 length_penalty: float = 0.0, portion: int = 512):
        vocab = stepper.vocab_size
        if width < 1 or max_tokens < 1:
            raise ValueError("beam search needs a width and a number of tokens of at least one")
        if min(2 * width, vocab) > kernels.MAX_ALTERNATIVES:
            raise ValueError(f"a beam search is at most {kernels.MAX_ALTERNATIVES // 2} beams wide")
        if not math.isfinite(length_penalty):
            raise ValueError("length_penalty must be finite")
        self.stepper, self.cache = stepper, stepper.cache
        self.width, self.max_tokens, self.end_ids = width, max_tokens, end_ids
        self.length_penalty, self.portion = length_penalty, max(1, portion)
        # Of a beam's first tokens as many may end it as there are ids that do, and behind them `width` may have to go on.  Where
        # that is more than one call ranks, those that go on are ranked by themselves as well.
        ends = sorted(t for t in end_ids if 0 <= t < vocab)
        listed = min(max(2 * width, width + len(ends)), vocab)
        self.top = min(listed, kernels.MAX_ALTERNATIVES)
        self._apart = ends if listed > self.top else []
        self._names = 0

    # ------------------------------------------------------------------ room
    def check(self, prompt: Sequence[int]) -> None:
        """Raise :class:`RequestRejected` for a prompt that the model or the whole cache cannot take at this width."""
        if not prompt:
            raise RequestRejected("the prompt is empty")
        if len(prompt) + self.max_tokens > self.stepper.max_positions:
            raise RequestRejected(f"prompt plus max_tokens ({len(prompt) + self.max_tokens}) exceeds the model's "
                                  f"{self.stepper.max_positions} positions")
        if self.width > self.cache.max_requests:
            raise RequestRejected(f"{self.width} beams need as many running requests ({self.cache.max_requests} at most)")
        for need, pool in self._needs(prompt):
            if need > pool.num_pages:
                raise RequestRejected(f"{self.width} beams behind a prompt of {len(prompt)} tokens need {need} cache pages of "
                                      f"{pool.num_pages}")

    def _needs(self, prompt: Sequence[int]):
        """Pages that a prompt and its beams may hold at once, per paged group."""
        total = len(prompt) + self.max_tokens
        pools = [g.pool for g in self.cache.groups if g.pool is not None]
        return [(shared + self.width * own, pool) for (shared, own), pool in zip(self.cache.fork_pages(len(prompt), total), pools)]

    def _fits(self, prompts: Sequence[Sequence[int]], slots: int, pages: Sequence[int]) -> bool:
        """Whether searches of these prompts, at their largest, fit ``slots`` requests and ``pages`` pages a group."""
        needs = [[need for need, _ in self._needs(prompt)] for prompt in prompts]
        return self.width * len(prompts) <= slots and all(sum(n) <= room for n, room in zip(zip(*needs), pages))

    def _name(self) -> Hashable:
        self._names += 1
        return ("beam", id(self), self._names)

    # ------------------------------------------------------------------ the search
    def run(self, prompts: Sequence[Sequence[int]]) -> List[List[BeamOutput]]:
        """The best ``width`` continuations of every prompt, best first.  Prompts run side by side as far as the cache has room."""
        for prompt in prompts:
            self.check(prompt)
        done: Dict[int, List[BeamOutput]] = {}
        waiting = list(enumerate(prompts))
        searches: List[_Search] = []
        # the room that this call may use: every search that runs keeps what it needs at its largest, so none stops half way
        slots = self.cache.slots.free_slots
        pages = [g.pool.available_to_reserve for g in self.cache.groups if g.pool is not None]
        try:
            while waiting or searches:
                while waiting and self._fits([search.prompt for search in searches] + [waiting[0][1]], slots, pages):
                    self._start(searches, *waiting.pop(0))
                if not searches:
                    raise RequestRejected("the cache has no room: other requests hold it")
                searches = self._advance(searches, done)
        finally:
            for search in searches:
                for beam in search.beams:
                    self.cache.release(beam.request)
        return [done[index] for index in range(len(prompts))]

    def _start(self, searches: List[_Search], index: int, prompt: Sequence[int]) -> None:
        cache, prompt = self.cache, list(prompt)
        request = self._name()
        if not cache.admit(request, reserve_tokens=len(prompt) + self.max_tokens):
            raise RequestRejected("the cache has no room: other requests hold it")
        logits = None
        try:
            for begin in range(0, len(prompt), self.portion):
                part = prompt[begin:begin + self.portion]
                last = begin + len(part) == len(prompt)
                logits = self.stepper.step([StepEntry(request, part, [len(part) - 1] if last else [])])
        except BaseException:
            cache.release(request)
            raise
        search = _Search(index, prompt, [_Beam(request, [], [], 0.0)])
        searches.append(search)                          # (whose beams go back to the cache whatever happens from here on)
        self._choose([search], self._alternatives(logits))

    def _alternatives(self, logits: torch.Tensor):
        """Per row: the most probable tokens and their log probabilities, on the host."""
        none = torch.zeros(logits.shape[0], dtype=torch.int32, device=logits.device)
        _, _, values, ids = kernels.token_logprobs(logits, none, self.top)
        ids, values = ids.tolist(), values.double().tolist()
        if not self._apart:
            return ids, values
        others = logits.index_fill(1, torch.tensor(self._apart, device=logits.device), -math.inf)
        best = kernels.token_logprobs(others, none, self.width)[3]
        logs = [kernels.token_logprobs(logits, column.contiguous())[0].double().tolist() for column in best.unbind(1)]
        for row, more in enumerate(best.tolist()):
            ranked = dict(zip(ids[row], values[row]))
            ranked.update((token, logs[k][row]) for k, token in enumerate(more))
            ids[row] = sorted(ranked, key=lambda token: (-ranked[token], token))
            values[row] = [ranked[token] for token in ids[row]]
        return ids, values

    def _advance(self, searches: List[_Search], done: Dict[int, List[BeamOutput]]) -> List[_Search]:
        """Close what is done, then one step of all beams of the others."""
        going: List[_Search] = []
        for search in searches:
            if search.beams and len(search.finished) < self.width and len(search.beams[0].tokens) < self.max_tokens:
                going.append(search)
                continue
            for beam in search.beams:
                self.cache.release(beam.request)
                if len(beam.tokens) >= self.max_tokens:
                    search.finished.append(self._output(beam.tokens, beam.logprobs, beam.total, FINISH_LENGTH))
            search.beams = []
            search.finished.sort(key=lambda out: -out.score)         # (stable: of equal scores the one found first)
            done[search.index] = search.finished[:self.width]
        if going:
            beams = [beam for search in going for beam in search.beams]
            logits = self._step([StepEntry(beam.request, [beam.tokens[-1]], [0]) for beam in beams])
            self._choose(going, self._alternatives(logits))
        return going

    def _step(self, entries: List[StepEntry]) -> torch.Tensor:
        graphs = self.stepper.graphs
        if graphs is not None and graphs.eligible(entries):
            zeros = [0.0] * len(entries)
            launch = graphs.launch(entries, zeros, zeros)
            return launch.graph.logits[:launch.count]
        return self.stepper.step(entries)

    def _output(self, tokens, logprobs, total, reason) -> BeamOutput:
        return BeamOutput(tokens, logprobs, _rank(total, len(tokens), self.length_penalty), reason)

    def _choose(self, searches: Sequence[_Search], alternatives) -> None:
        """The continuations that go on, from every beam's most probable tokens (rows in the order of the searches' beams)."""
        ids, values = alternatives
        row, found, forks, released = 0, [], [], []
        for search in searches:
            candidates = []
            for place, beam in enumerate(search.beams):
                for rank, (token, value) in enumerate(zip(ids[row], values[row])):
                    if value > -math.inf:                            # (a token that the model rules out, or NaN, is no continuation)
                        candidates.append((-(beam.total + value), place, rank, token, value))
                row += 1
            if not candidates:
                raise InvalidLogits("beam search received logits that give no token a probability")
            found.append(sorted(candidates))
        for search, candidates in zip(searches, found):
            chosen: List[Tuple[int, int, float, float]] = []
            for position, (negative, place, _, token, value) in enumerate(candidates):
                if len(chosen) == self.width:
                    break
                beam = search.beams[place]
                if token in self.end_ids:
                    if position < self.width:                        # (one that ends counts where it is among the best itself)
                        search.finished.append(self._output(beam.tokens + [token], beam.logprobs + [value], -negative, FINISH_STOP))
                    continue
                chosen.append((place, token, value, -negative))
            taken: Dict[int, bool] = {}
            beams = []
            for place, token, value, total in chosen:
                beam = search.beams[place]
                request = beam.request
                if place in taken:
                    request = self._name()
                    forks.append((search, beam.request, request))
                taken[place] = True
                beams.append(_Beam(request, beam.tokens + [token], beam.logprobs + [value], total))
            released += [beam.request for place, beam in enumerate(search.beams) if place not in taken]
            search.beams = beams
        for request in released:
            self.cache.release(request)
        if not self.cache.fork([(parent, child) for _, parent, child in forks],
                               [len(search.prompt) + self.max_tokens for search, _, _ in forks]):
            raise RequestRejected("the cache has no room for the beams: other requests hold it")


def score(stepper: Stepper, sequence: Sequence[int], alternatives: int = 0, portion: int = 512) -> TokenScores:
    """The model's log probabilities of a given sequence, portion by portion."""
    sequence = [int(t) for t in sequence]
    if not sequence:
        raise RequestRejected("the sequence is empty")
    if not 0 <= sequence[-1] < stepper.vocab_size:                   # (which no step runs)
        raise StepError(f"token id {sequence[-1]} is outside the vocabulary of {stepper.vocab_size}")
    if len(sequence) > stepper.max_positions:
        raise RequestRejected(f"the sequence has {len(sequence)} tokens, the model {stepper.max_positions} positions")
    request = ("score", id(sequence))
    cache = stepper.cache
    out = TokenScores(sequence, [], [])
    if len(sequence) == 1:
        return out
    if not cache.admit(request, reserve_tokens=len(sequence)):
        raise RequestRejected(f"the cache has no room for a sequence of {len(sequence)} tokens")
    try:
        # (the last token is nobody's condition)
        for begin in range(0, len(sequence) - 1, portion):
            part = sequence[begin:min(begin + portion, len(sequence) - 1)]
            logits = stepper.step([StepEntry(request, part, list(range(len(part))))])
            following = torch.tensor(sequence[begin + 1:begin + 1 + len(part)], dtype=torch.int32, device=logits.device)
            logprob, entropy, values, ids = kernels.token_logprobs(logits, following, alternatives)
            out.logprobs += logprob.tolist()
            out.entropies += entropy.tolist()
            if alternatives:
                out.alternatives += [list(zip(i, v)) for i, v in zip(ids.tolist(), values.tolist())]
    finally:
        cache.release(request)
    return out
