"""How a step chooses the tokens of its rows, up to the kernels (no device): a step function whose sampler is a stand-in."""

from types import SimpleNamespace

import numpy as np
import pytest
import torch

import tesseract_b200.parts  # noqa: F401
from tesseract_b200 import kernels
from tesseract_b200.cache import CacheManager
from tesseract_b200.engine.step import StepEntry, Stepper
from tesseract_b200.parts import PagedKVNeed
from tesseract_b200.sampling import SamplingParams
from tesseract_b200.sampling.params import TokenChoice
from tests import token_choice_plain as plain


def make_stepper(requests, vocab=100, model=None):
    cache = CacheManager([PagedKVNeed(2, 16)], [None], num_pages=64, page_size=16, max_requests=len(requests), dtype=torch.float32,
                         device="cpu", max_step_tokens=64, allocate_storage=False)
    for request in requests:
        assert cache.admit(request)
    made = SimpleNamespace(runtime=SimpleNamespace(device=torch.device("cpu")), spec=SimpleNamespace(vocab_size=vocab, max_positions=256))
    if model is not None:
        made.forward = model
    return Stepper(made, cache)


class Told:
    """A sampler that keeps what it is asked."""

    def __init__(self):
        self.sampled, self.chosen = [], []

    def sample(self, logits, temperatures, top_ps, draws):
        self.sampled.append(dict(rows=logits.shape[0], temperatures=list(temperatures), top_ps=list(top_ps), draws=list(draws)))
        return [5] * logits.shape[0]

    def choose(self, logits, temperatures, draws, **given):
        self.chosen.append(dict(rows=logits.shape[0], temperatures=list(temperatures), draws=list(draws), **given))
        return [6] * logits.shape[0]


@pytest.mark.parametrize("vocab", [kernels.MAX_CHOICE_VOCAB, kernels.MAX_CHOICE_VOCAB + 1])
def test_top_p_beyond_the_kernels_vocabulary_goes_to_the_hosts_sampler(vocab):
    """A step that is not captured: the one in which a prompt ends, whose row stands beside others."""
    stepper = make_stepper("abc", vocab)
    stepper._sampler = told = Told()
    stepper.step = lambda entries: torch.zeros(3, 8)
    cut, greedy = SamplingParams(top_p=0.5), SamplingParams(temperature=0.0)
    entries = [StepEntry("a", [1, 2], [1], TokenChoice.of(cut, 2)), StepEntry("b", [3], [0], TokenChoice.of(greedy, 1)), StepEntry("c", [4], [0])]
    tokens = stepper.step_and_sample(entries, [1.0, 0.0, 0.7], [0.5, 1.0, 1.0], [0.1, 0.2, 0.3])
    given = (told.chosen if vocab <= kernels.MAX_CHOICE_VOCAB else told.sampled)
    assert len(told.chosen) + len(told.sampled) == 1 and len(given) == 1 and len(tokens) == 3
    assert given[0]["rows"] == 3 and given[0]["top_ps"] == [0.5, 1.0, 1.0] and given[0]["draws"] == [0.1, 0.2, 0.3]


def test_rows_that_nothing_is_said_of_are_marked():
    """Beside rows with rules and cuts they keep the sampler's token whatever their logits are."""
    kinds = [SamplingParams(), SamplingParams(temperature=0.0, top_p=0.5, top_k=3, min_p=0.1), SamplingParams(top_p=0.5),
             SamplingParams(top_k=4), SamplingParams(min_p=0.2), SamplingParams(temperature=0.0, presence_penalty=1.0)]
    stepper = make_stepper(range(len(kinds)))
    stepper._sampler = told = Told()
    stepper._rules = object()
    stepper.step = lambda entries: torch.zeros(len(kinds), 8)
    entries = [StepEntry(i, [1], [0], TokenChoice.of(params, 1)) for i, params in enumerate(kinds)]
    stepper.step_and_sample(entries, [p.temperature for p in kinds], [p.top_p for p in kinds], [0.5] * len(kinds))
    assert told.chosen[0]["as_sampled"] == [True, True, False, False, False, False]
    assert [TokenChoice.plain(e.choice, p.temperature, p.top_p) for e, p in zip(entries, kinds)] == [True, True, False, False, False, False]
    # (top-p may come without a choice)
    assert not TokenChoice.plain(None, 1.0, 0.5) and TokenChoice.plain(None, 0.0, 0.5) and TokenChoice.plain(None, 1.0, 1.0)


class Noted:
    """Histories on the host in place of the kernel's, and what was asked for them."""

    def __init__(self, monkeypatch, slots, vocab=100):
        self.seen, self.counts, self.calls = np.zeros((slots, vocab), dtype=bool), np.zeros((slots, vocab), dtype=np.int64), []
        monkeypatch.setattr(kernels, "note_tokens", self.note)

    def note(self, rules, slots, tokens, *, starts=None, prompts=None, restart=False):
        slots, tokens, starts = slots.tolist(), tokens.tolist(), starts.tolist()
        prompts = [0] * len(slots) if prompts is None else prompts.tolist()
        self.calls.append((slots, [tokens[a:b] for a, b in zip(starts, starts[1:])], prompts, restart))
        for slot, part, prompt in zip(*self.calls[-1][:3]):
            plain.note(self.seen, self.counts, slot, part, prompt, restart)


class OnHost:
    """The staging of arrays without a device."""

    @staticmethod
    def upload(arrays):
        return [torch.from_numpy(np.ascontiguousarray(a).copy()) for a in arrays]


def noting_stepper(monkeypatch, requests, forward):
    stepper = make_stepper(requests, model=forward)
    stepper._staging = OnHost
    return stepper, Noted(monkeypatch, stepper.cache.max_requests)


def test_a_step_that_fails_leaves_histories_as_they_were(monkeypatch):
    """Tried again it brings its tokens once."""
    failing = []

    def forward(*args, **kwargs):
        if failing:
            raise RuntimeError(failing.pop())
        return torch.zeros(1, 100)

    stepper, noted = noting_stepper(monkeypatch, "ab", forward)
    slot = stepper.cache.slot("a")
    choice = TokenChoice.of(SamplingParams(frequency_penalty=0.5), 3)
    for tokens in ([5, 6], [7], [8], [8], [9]):                        # (a prompt of three, then its answer)
        before = noted.seen.copy(), noted.counts.copy()
        failing.append("injected")
        with pytest.raises(RuntimeError, match="injected"):
            stepper.step([StepEntry("a", tokens, [], choice)])
        assert np.array_equal(noted.seen, before[0]) and np.array_equal(noted.counts, before[1])
        stepper.step([StepEntry("a", tokens, [], choice)])
    assert np.flatnonzero(noted.seen[slot]).tolist() == [5, 6, 7, 8, 9]
    assert noted.counts[slot, [5, 6, 7, 8, 9]].tolist() == [0, 0, 0, 2, 1] and noted.counts.sum() == 3
    # pages that run out in the middle of a step
    stepper.cache.extend("b", 49 * 16)
    before = noted.counts.copy()
    with pytest.raises(Exception, match="(?i)pages"):
        stepper.step([StepEntry("a", [3] * 241, [], choice)])
    assert np.array_equal(noted.counts, before) and not noted.seen[slot, 3]


def test_a_request_that_begins_has_its_tokens_in_place_of_what_its_slot_had(monkeypatch):
    """One call for the requests that begin with a step and one for the others, and none for those without penalties."""
    stepper, noted = noting_stepper(monkeypatch, "abc", lambda *args, **kwargs: torch.zeros(3, 100))
    slot = {request: stepper.cache.slot(request) for request in "abc"}
    noted.seen[:], noted.counts[:] = True, 7                           # (slots that others had)
    penalised, biased = SamplingParams(presence_penalty=0.5), SamplingParams(logit_bias={3: 1.0})
    choice = {"a": TokenChoice.of(penalised, 3), "b": TokenChoice.of(biased, 2), "c": TokenChoice.of(penalised, 1)}
    stepper.step([StepEntry("a", [5, 6], [], choice["a"]), StepEntry("b", [9, 9], [], choice["b"])])
    assert noted.calls == [([slot["a"]], [[5, 6]], [3], True)]
    stepper.step([StepEntry("a", [7, 8], [], choice["a"]), StepEntry("c", [4, 4, 4], [], choice["c"])])
    assert noted.calls[1:] == [([slot["c"]], [[4, 4, 4]], [1], True), ([slot["a"]], [[7, 8]], [1], False)]
    stepper.step([StepEntry("c", [4], [], choice["c"]), StepEntry("a", [8], [], choice["a"]), StepEntry("b", [1], [], choice["b"])])
    assert noted.calls[3:] == [([slot["c"], slot["a"]], [[4], [8]], [-2, -1], False)]
    assert np.flatnonzero(noted.seen[slot["a"]]).tolist() == [5, 6, 7, 8] and noted.counts[slot["a"], 8] == 2
    assert noted.counts[slot["a"]].sum() == 2 and noted.counts[slot["c"], 4] == 3 and noted.counts[slot["c"]].sum() == 3
    # in front of a captured step, which notes what it is fed
    stepper.cache.release("a")
    assert stepper.cache.admit("d")
    stepper.begin_histories([StepEntry("d", [5], [0], choice["a"]), StepEntry("c", [5], [0], choice["c"]), StepEntry("b", [1], [0], choice["b"])])
    assert noted.calls[4:] == [([stepper.cache.slot("d")], [[]], [3], True)] and not noted.seen[stepper.cache.slot("d")].any()


def test_the_table_of_rules_is_made_on_demand_and_once():
    stepper = make_stepper("ab")
    assert stepper._rules is None
    stepper.prepare_rules()
    rules = stepper._rules
    assert rules.slots == stepper.cache.max_requests and rules.vocab == 100
    stepper.prepare_rules()
    assert stepper._rules is rules and stepper.rules is rules
