"""Beam search and scoring over a stand-in model, against a search written without a cache (no GPU needed)."""

import hashlib
import math
import types

import numpy as np
import pytest
import torch

import tesseract_b200.parts  # noqa: F401
from tesseract_b200.cache import CacheManager
from tesseract_b200.engine.beam import BeamSearch, TokenScores, score
from tesseract_b200.engine.scheduler import RequestRejected
from tesseract_b200.parts import PagedKVNeed, StateNeed
from tesseract_b200.sampling import InvalidLogits

VOCAB = 23


def logits_of(tokens):
    """A row of logits that depends on every token in front of it and their order."""
    seed = int.from_bytes(hashlib.sha256(bytes(tokens)).digest()[:4], "little")
    return np.random.RandomState(seed).standard_normal(VOCAB) * 2.0


def log_softmax(x):
    m = x.max()
    return x - m - math.log(np.exp(x - m).sum())


class FakeStepper:
    """Runs the cache as the step function does; what a request has seen it knows from the pages that its block table names."""

    graphs = None
    vocab_size = VOCAB

    def __init__(self, needs=None, num_pages=200, page_size=4, max_requests=16, max_positions=200, logits=logits_of):
        needs = needs or [PagedKVNeed(1, 1)]
        self.cache = CacheManager(needs, [None] * len(needs), num_pages=num_pages, page_size=page_size, max_requests=max_requests,
                                  dtype=torch.float32, device="cpu", max_step_tokens=8)
        self.max_positions, self.logits = max_positions, logits
        self.rows = []

    def step(self, entries):
        out = []
        self.rows.append(len(entries))
        storage = self.cache.groups[0].storage.view(1, -1, 2, self.cache.page_size)
        for entry in entries:
            begin, count = self.cache.length(entry.request), len(entry.tokens)
            self.cache.extend(entry.request, count)
            pages = self.cache.block_table_rows(0, [self.cache.slot(entry.request)], 64)[0]
            for k, token in enumerate(entry.tokens):
                position = begin + k
                storage[0, int(pages[position // self.cache.page_size]), 0, position % self.cache.page_size] = float(token)
            seen = [int(storage[0, int(pages[i // self.cache.page_size]), 0, i % self.cache.page_size]) for i in range(begin + count)]
            out += [self.logits(seen[:begin + place + 1]) for place in entry.want]
            self.cache.commit(entry.request, count)
        self.cache.check()
        return torch.tensor(np.array(out)) if out else None


class HostSearch(BeamSearch):
    def _alternatives(self, logits):
        logs = torch.log_softmax(logits.double(), dim=-1)
        values, ids = torch.sort(logs, dim=-1, descending=True, stable=True)
        return ids[:, :self.top].tolist(), values[:, :self.top].tolist()


def plain_search(prompt, width, max_tokens, ends, penalty, logits=logits_of):
    beams, finished = [([], 0.0)], []
    while beams and len(finished) < width and len(beams[0][0]) < max_tokens:
        every = []
        for place, (tokens, total) in enumerate(beams):
            logs = log_softmax(logits(list(prompt) + tokens))
            order = sorted(range(VOCAB), key=lambda t: (-logs[t], t))[:min(2 * width, VOCAB)]
            every += [(-(total + logs[t]), place, rank, t) for rank, t in enumerate(order)]
        every.sort()
        new = []
        for position, (negative, place, _, token) in enumerate(every):
            if len(new) == width:
                break
            if token in ends:
                if position < width:
                    finished.append((beams[place][0] + [token], -negative))
            else:
                new.append((beams[place][0] + [token], -negative))
        beams = new
    if beams and len(beams[0][0]) >= max_tokens:
        finished += beams
    finished = [(tokens, total / len(tokens) ** penalty) for tokens, total in finished]
    return sorted(finished, key=lambda f: -f[1])[:width]


@pytest.mark.parametrize("width", [1, 2, 4, 7])
@pytest.mark.parametrize("penalty", [0.0, 1.0])
@pytest.mark.parametrize("ends", [(), (3,), (3, 8, 11, 20)])
def test_finds_what_a_search_without_a_cache_finds(width, penalty, ends):
    prompts = [[1, 2, 3, 4, 5], [7], list(range(13)), [9, 9, 9, 9]]
    stepper = FakeStepper(max_requests=16)
    found = HostSearch(stepper, width, 9, end_ids=frozenset(ends), length_penalty=penalty, portion=4).run(prompts)
    for prompt, outs in zip(prompts, found):
        want = plain_search(prompt, width, 9, set(ends), penalty)
        assert [o.token_ids for o in outs] == [tokens for tokens, _ in want]
        for out, (tokens, value) in zip(outs, want):
            assert out.score == pytest.approx(value, abs=1e-9)
            assert out.logprob == pytest.approx(value * len(tokens) ** penalty, abs=1e-9)
            assert out.finish_reason == ("stop" if tokens[-1] in ends else "length")
    assert stepper.cache.used_pages() == 0 and stepper.cache.slots.free_slots == 16
    stepper.cache.check()


def test_prompts_wait_where_the_cache_has_no_room_for_them():
    stepper = FakeStepper(num_pages=20, max_requests=6)
    prompts = [[k] * 6 for k in range(5)]                  # 1 shared page + 3 beams of 3 of their own: ten pages a prompt
    found = HostSearch(stepper, 3, 8, portion=8).run(prompts)
    for prompt, outs in zip(prompts, found):
        assert [o.token_ids for o in outs] == [tokens for tokens, _ in plain_search(prompt, 3, 8, set(), 0.0)]
    assert max(stepper.rows) == 6                          # two prompts side by side
    assert stepper.cache.used_pages() == 0


def test_windows_and_states_fork_too():
    stepper = FakeStepper([PagedKVNeed(1, 1), PagedKVNeed(1, 1, 5), StateNeed((4,))])
    found = HostSearch(stepper, 4, 10, portion=8).run([[1, 2, 3], [4] * 11])
    for prompt, outs in zip([[1, 2, 3], [4] * 11], found):
        assert [o.token_ids for o in outs] == [tokens for tokens, _ in plain_search(prompt, 4, 10, set(), 0.0)]
    assert stepper.cache.used_pages() == 0


def test_refusals():
    stepper = FakeStepper(num_pages=20, max_requests=4, max_positions=50)
    for width, tokens in ((0, 3), (2, 0), (33, 3)):
        big = types.SimpleNamespace(vocab_size=1000, cache=stepper.cache, max_positions=50)
        with pytest.raises(ValueError):
            BeamSearch(big, width, tokens)
    with pytest.raises(ValueError):
        BeamSearch(stepper, 2, 3, length_penalty=math.nan)
    for width, tokens, prompt in [(2, 5, []), (5, 5, [1]), (2, 45, [1] * 10), (4, 30, [1] * 8)]:
        with pytest.raises(RequestRejected):
            HostSearch(stepper, width, tokens).run([[1, 2], prompt])
    assert stepper.cache.used_pages() == 0                 # nothing had begun
    stepper.cache.admit("someone", reserve_tokens=60)
    with pytest.raises(RequestRejected, match="no room"):
        HostSearch(stepper, 2, 20).run([[1] * 8])
    assert stepper.cache.slots.free_slots == 3


@pytest.mark.parametrize("sequence", [[], [1, 2, VOCAB], [1, 2, -1], [VOCAB], [1] * 51])
def test_scoring_refuses_what_no_step_would_run(sequence):
    stepper = FakeStepper(max_positions=50)
    with pytest.raises((RequestRejected, ValueError)):
        score(stepper, sequence)
    assert stepper.cache.used_pages() == 0 and stepper.cache.slots.free_slots == 16 and not stepper.rows


def test_logits_without_a_probability_fail_and_leave_nothing_behind():
    def broken(tokens):
        return logits_of(tokens) if len(tokens) < 6 or tokens[0] != 2 else np.full(VOCAB, np.nan)

    stepper = FakeStepper(logits=broken)
    with pytest.raises(InvalidLogits):
        HostSearch(stepper, 3, 8).run([[1, 2, 3], [2, 3, 4]])
    assert stepper.cache.used_pages() == 0 and stepper.cache.slots.free_slots == 16
    stepper.cache.check()


def test_fewer_tokens_than_beams():
    def narrow(tokens):
        row = np.full(VOCAB, -np.inf)
        row[:2] = [0.3, 0.1 * (len(tokens) % 3)]
        return row

    found = HostSearch(FakeStepper(logits=narrow), 6, 4).run([[5]])[0]
    assert len(found) == 6 and len({tuple(o.token_ids) for o in found}) == 6
    assert [o.score for o in found] == sorted((o.score for o in found), reverse=True)


def test_perplexity_of_nothing_and_of_something():
    assert TokenScores([1], [], []).perplexity == 1.0
    assert TokenScores([1, 2, 3], [math.log(0.5), math.log(0.125)], [0.0, 0.0]).perplexity == pytest.approx(4.0)


def whole_search(prompt, width, max_tokens, ends, logits):
    """The same with every token of every beam ranked: the best `width` that go on, and those that end among the best `width`."""
    beams, finished = [([], 0.0)], []
    while beams and len(finished) < width and len(beams[0][0]) < max_tokens:
        every = []
        for place, (tokens, total) in enumerate(beams):
            logs = log_softmax(logits(list(prompt) + tokens))
            order = sorted(range(VOCAB), key=lambda t: (-logs[t], t))
            every += [(-(total + logs[t]), place, rank, t) for rank, t in enumerate(order)]
        every.sort()
        finished += [(beams[place][0] + [t], -negative) for negative, place, _, t in every[:width] if t in ends]
        beams = [(beams[place][0] + [t], -negative) for negative, place, _, t in every if t not in ends][:width]
    if beams and len(beams[0][0]) >= max_tokens:
        finished += beams
    return sorted(finished, key=lambda f: -f[1])[:width]


@pytest.mark.parametrize("width, ends", [(2, (1, 4, 9)), (2, tuple(range(2, 12))), (3, (0, 5, 6, 7, 8, 20)), (4, tuple(range(6, 20))),
                                         (5, (3, 4, 30, -1, 7, 9, 10, 11))])
def test_many_ids_that_end_a_beam_leave_the_others_their_places(width, ends):
    """Where most of a beam's best tokens end it, its next ones go on all the same."""
    valid = [t for t in ends if 0 <= t < VOCAB]
    others = [t for t in range(VOCAB) if t not in ends]

    def ending(tokens):
        row = 0.01 * logits_of(tokens)
        if len(tokens) == 3:                                   # first: one that goes on, all that end, then the others
            row[valid] += 4.5
            row[others] += 4.0
            row[others[0]] += 1.0
        elif tokens[3] != others[0]:                           # (the others' next token is certain, the first one's is not)
            row[others[tokens[0] % len(others)]] += 20.0
        return row

    stepper = FakeStepper(logits=ending)
    prompts = [[k, 2 * k % VOCAB, 5] for k in range(12)]
    shorter = 0
    for prompt, outs in zip(prompts, HostSearch(stepper, width, 7, end_ids=frozenset(ends)).run(prompts)):
        want = whole_search(prompt, width, 7, set(ends), ending)
        assert [o.token_ids for o in outs] == [tokens for tokens, _ in want]
        assert [o.score for o in outs] == pytest.approx([value for _, value in want], abs=1e-9)
        shorter += [t for t, _ in plain_search(prompt, width, 7, set(ends), 0.0, ending)] != [t for t, _ in want]
    assert shorter                                         # (twice the width of a beam's tokens is not enough for these)
