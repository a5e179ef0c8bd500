"""What a request says about its next tokens, up to the step function (no GPU needed): options and their refusals, what the scheduler
hands on, grammars, and requests that no token can follow."""

import math

import numpy as np
import pytest

from tesseract_b200.config.engine_config import EngineConfig
from tesseract_b200.engine.scheduler import FINISH_ERROR, FINISH_LENGTH, RequestRejected, Scheduler
from tesseract_b200.sampling import SamplingParams
from tesseract_b200.sampling.params import TokenChoice
from tests.test_scheduler import FakeAheadEngine, run_all


@pytest.mark.parametrize("given", [
    dict(top_k=-1), dict(top_k=1.5), dict(top_k=2 ** 31), dict(min_p=-0.1), dict(min_p=1.1), dict(min_p=math.nan),
    dict(repetition_penalty=0.0), dict(repetition_penalty=-1.0), dict(repetition_penalty=math.inf), dict(presence_penalty=math.nan),
    dict(frequency_penalty=math.inf), dict(logit_bias={-1: 1.0}), dict(logit_bias={"a": 1.0}), dict(logit_bias={1: math.nan}),
    dict(logit_bias={1: math.inf}), dict(logit_bias={t: 1.0 for t in range(1025)}), dict(allowed_token_ids=[]),
    dict(allowed_token_ids=[-1]), dict(allowed_token_ids=[0.5]), dict(grammar=7),
    # (what the kernels' 32 bits do not hold)
    dict(logit_bias={1: 1e39}), dict(repetition_penalty=1e39), dict(repetition_penalty=1e-60), dict(presence_penalty=-1e39),
    dict(frequency_penalty=1e39)], ids=str)
def test_options_that_are_refused(given):
    with pytest.raises(ValueError):
        SamplingParams(**given)


def test_options_are_kept_as_numbers():
    params = SamplingParams(logit_bias={True: 2, np.int64(7): np.float32(0.5), 9: -1e39}, allowed_token_ids=np.asarray([True, False]).tolist())
    assert params.logit_bias == {1: 2.0, 7: 0.5, 9: -1e39} and params.allowed_token_ids == (1, 0)
    assert [type(token) for token in (*params.logit_bias, *params.allowed_token_ids)] == [int] * 5
    assert [type(bias) for bias in params.logit_bias.values()] == [float] * 3


def test_which_options_are_rules_and_which_are_cuts():
    assert TokenChoice.of(SamplingParams(), 3) is None and TokenChoice.of(SamplingParams(temperature=0.0, top_p=0.5, top_k=4), 3) is None
    for given in (dict(top_p=0.9), dict(top_k=3), dict(min_p=0.1)):
        choice = TokenChoice.of(SamplingParams(**given), 3)
        assert choice.params.cut and not choice.params.ruled and choice.prompt_tokens == 3
    for given in (dict(repetition_penalty=1.1), dict(presence_penalty=-0.5), dict(frequency_penalty=0.5), dict(logit_bias={3: -math.inf}),
                  dict(allowed_token_ids=[1]), dict(grammar=lambda tokens: [1])):
        params = SamplingParams(temperature=0.0, **given)
        assert params.ruled and not params.cut and TokenChoice.of(params, 3) is not None
        assert params.penalised == any(name.endswith("_penalty") for name in given)
    assert not SamplingParams(logit_bias={}).ruled
    with pytest.raises(ValueError):
        SamplingParams(logit_bias={100: 1.0}).check_vocabulary(100)
    with pytest.raises(ValueError):
        SamplingParams(allowed_token_ids=[3, 100]).check_vocabulary(100)
    SamplingParams(logit_bias={99: 1.0}, allowed_token_ids=[99]).check_vocabulary(100)


class Choosing(FakeAheadEngine):
    """The fake, which keeps the choices that it is given and looks at masks: the token that would follow, if it is allowed."""

    def __init__(self, config, **kw):
        super().__init__(config, **kw)
        self.choices, self.ruled_out = [], set()

    def can_launch_decode(self, rows, top_ps):
        return 0 < rows <= 4

    def _follow(self, entry, last):
        token = 1000 if last < 1000 else last + 1
        self.choices.append((entry.request, entry.choice))
        allowed = entry.choice.allowed if entry.choice is not None else None
        if allowed is not None and not int(allowed[token // 32]) >> token % 32 & 1 or token in self.ruled_out:
            return -1
        return token

    def run_and_sample(self, entries, temperatures, top_ps, draws):
        wanted = [e for e in entries if e.want]
        return [self._follow(e, row) for e, row in zip(wanted, self.run_step(entries))]

    def launch_decode(self, entries, temperatures, draws, previous, fed):
        launch = super().launch_decode(entries, temperatures, draws, previous, fed)
        launch._tokens = [self._follow(e, token - 1 if token > 1000 else 0) for e, token in zip(entries, launch._tokens)]
        return launch


def make(vocab=2000, ahead=True, **kw):
    config = EngineConfig(max_queue=8, max_running=4, max_batch_tokens=32, prefill_chunk_tokens=8,
                          kv_capacity_tokens=512, max_sequence_length=512)
    fake = Choosing(config, **kw)
    scheduler = Scheduler(config, fake.cache, fake.run_step, fake.sample, max_positions=400, run_and_sample=fake.run_and_sample,
                          launch_decode=fake.launch_decode if ahead else None,
                          can_launch_decode=fake.can_launch_decode if ahead else None, vocab_size=vocab)
    return scheduler, fake


def test_a_token_outside_the_vocabulary_is_refused_when_the_request_arrives():
    s, _ = make()
    for given in (dict(logit_bias={2000: 1.0}), dict(allowed_token_ids=[1, 5000])):
        with pytest.raises(ValueError):
            s.add_request([1, 2], SamplingParams(**given))
    assert not s.has_work()


def test_a_scheduler_whose_sampler_takes_no_rules_refuses_them():
    config = EngineConfig(max_queue=8, max_running=4, max_batch_tokens=32, prefill_chunk_tokens=8,
                          kv_capacity_tokens=512, max_sequence_length=512)
    fake = Choosing(config)
    plain = Scheduler(config, fake.cache, fake.run_step, fake.sample, max_positions=400)
    for given in (dict(top_k=4), dict(min_p=0.1), dict(logit_bias={3: 1.0}), dict(grammar=lambda tokens: [1])):
        with pytest.raises(RequestRejected):
            plain.add_request([1, 2], SamplingParams(**given))
    plain.add_request([1, 2], SamplingParams(max_tokens=2, top_p=0.5))


def test_a_vocabulary_beyond_the_kernels_takes_no_rules():
    """A request that a step could only fail with all that stand beside it is refused at once."""
    config = EngineConfig(max_queue=8, max_running=4, max_batch_tokens=32, prefill_chunk_tokens=8,
                          kv_capacity_tokens=512, max_sequence_length=512)
    fake = Choosing(config)
    for vocab, taken in ((262144, True), (262145, False)):
        s = Scheduler(config, fake.cache, fake.run_step, fake.sample, max_positions=400, run_and_sample=fake.run_and_sample, vocab_size=vocab)
        for given in (dict(top_k=4), dict(min_p=0.1), dict(logit_bias={3: 1.0}), dict(grammar=lambda tokens: [1])):
            if taken:
                s.add_request([1, 2], SamplingParams(**given))
            else:
                with pytest.raises(RequestRejected):
                    s.add_request([1, 2], SamplingParams(**given))
        s.add_request([1, 2], SamplingParams(max_tokens=2, top_p=0.5))


@pytest.mark.parametrize("ahead", [False, True])
def test_choices_travel_with_the_steps(ahead):
    s, fake = make(ahead=ahead)
    ruled = SamplingParams(max_tokens=5, temperature=0.0, repetition_penalty=1.3, ignore_eos=True)
    a = s.add_request(list(range(11)), ruled)
    b = s.add_request([3], SamplingParams(max_tokens=5, temperature=0.0, ignore_eos=True))
    c = s.add_request([4, 5], SamplingParams(max_tokens=3, top_p=0.5, ignore_eos=True))
    done = {r.id: r for r in run_all(s)}
    assert [len(done[i].generated) for i in (a, b, c)] == [5, 5, 3] and (len(fake.launches) > 0) == ahead
    for request, choice in fake.choices:
        if request == a:
            assert choice.params is ruled and choice.prompt_tokens == 11 and choice.allowed is None
        elif request == b:
            assert choice is None
        else:
            assert choice.params.top_p == 0.5 and not choice.params.ruled


def test_a_grammar_is_asked_with_the_tokens_so_far_in_front_of_every_token():
    s, fake = make()
    asked = []

    def grammar(tokens):
        asked.append(list(tokens))
        return range(1000, 1100)

    a = s.add_request(list(range(20)), SamplingParams(max_tokens=4, temperature=0.0, grammar=grammar, ignore_eos=True,
                                                      allowed_token_ids=[1000, 1001, 1002, 1003, 7]))
    b = s.add_request([3], SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True))
    done = {r.id: r for r in run_all(s)}
    assert done[a].generated == [1000, 1001, 1002, 1003] and done[a].finish_reason == FINISH_LENGTH
    assert asked == [[], [1000], [1000, 1001], [1000, 1001, 1002]]
    assert len(done[b].generated) == 6
    masks = [choice.allowed for request, choice in fake.choices if request == a]
    for words in masks:
        assert [t for t in range(2000) if int(words[t // 32]) >> t % 32 & 1] == [1000, 1001, 1002, 1003]


def test_a_grammar_may_return_truth_values():
    s, fake = make()
    allowed = np.zeros(2000, dtype=bool)
    allowed[1000:1003] = True
    a = s.add_request([1, 2], SamplingParams(max_tokens=9, temperature=0.0, grammar=lambda tokens: allowed, ignore_eos=True))
    done = {r.id: r for r in run_all(s)}
    assert done[a].generated == [1000, 1001, 1002] and done[a].finish_reason == FINISH_ERROR


def test_a_grammar_that_fails_ends_its_request_alone():
    s, fake = make()

    def broken(tokens):
        if len(tokens) == 2:
            raise KeyError("no such state")
        return range(2000)

    a = s.add_request([1, 2], SamplingParams(max_tokens=9, temperature=0.0, grammar=broken, ignore_eos=True))
    b = s.add_request([1, 2], SamplingParams(max_tokens=9, temperature=0.0, grammar=lambda tokens: [2000], ignore_eos=True))
    c = s.add_request([3], SamplingParams(max_tokens=5, temperature=0.0, ignore_eos=True))
    done = {r.id: r for r in run_all(s)}
    assert done[a].finish_reason == FINISH_ERROR and "no such state" in done[a].error and done[a].generated == [1000, 1001]
    assert done[b].finish_reason == FINISH_ERROR and "vocabulary" in done[b].error and done[b].generated == []
    assert len(done[c].generated) == 5 and done[c].finish_reason == FINISH_LENGTH
    fake.cache.check()


@pytest.mark.parametrize("ahead", [False, True])
def test_a_request_that_no_token_can_follow_ends_with_those_it_has(ahead):
    s, fake = make(ahead=ahead)
    fake.ruled_out = {1003}
    a = s.add_request([5, 6, 7], SamplingParams(max_tokens=30, temperature=0.0, presence_penalty=1.0, ignore_eos=True))
    done = {r.id: r for r in run_all(s)}
    assert done[a].finish_reason == FINISH_ERROR and done[a].generated == [1000, 1001, 1002]
    assert "no token" in done[a].error
    b = s.add_request([5, 6, 7], SamplingParams(max_tokens=2, temperature=0.0, ignore_eos=True))       # (the engine goes on)
    assert {r.id: r for r in run_all(s)}[b].finish_reason == FINISH_LENGTH
    fake.cache.check()


def test_command_line_options(monkeypatch):
    from tesseract_b200 import cli

    args = cli.build_parser().parse_args(["--top-k", "40", "--min-p", "0.05", "--repetition-penalty", "1.2", "--presence-penalty", "0.5",
                                          "--frequency-penalty", "0.25", "--logit-bias", "5:-2.5,7:1", "--allowed-token-ids", "5,7,9"])
    params = cli.sampling_params(args)
    assert (params.top_k, params.min_p, params.repetition_penalty) == (40, 0.05, 1.2)
    assert (params.presence_penalty, params.frequency_penalty) == (0.5, 0.25)
    assert params.logit_bias == {5: -2.5, 7: 1.0} and params.allowed_token_ids == (5, 7, 9)
    assert not cli.sampling_params(cli.build_parser().parse_args([])).ruled


def test_a_request_whose_rules_have_no_room_is_refused_alone():
    """The table of rules is made when a request that needs it arrives: no step fails for want of it."""
    s, _ = make()
    asked = []

    def no_room():
        asked.append(len(s.requests))
        raise MemoryError("nothing left on the device")

    s.prepare_rules = no_room
    a = s.add_request([1, 2], SamplingParams(max_tokens=3, temperature=0.0, ignore_eos=True))
    b = s.add_request([3], SamplingParams(max_tokens=3, top_p=0.5, top_k=4, ignore_eos=True))          # (a cut needs none)
    assert asked == []
    with pytest.raises(RequestRejected, match="nothing left on the device"):
        s.add_request([1, 2], SamplingParams(max_tokens=3, presence_penalty=1.0))
    with pytest.raises(RequestRejected, match="capacity"):                                             # (nor one that is refused anyway)
        s.add_request([1, 2], SamplingParams(max_tokens=3000, presence_penalty=1.0))
    assert asked == [2] and len(s.requests) == 2
    s.prepare_rules = lambda: asked.append("made")
    c = s.add_request([1, 2], SamplingParams(max_tokens=3, temperature=0.0, presence_penalty=1.0, ignore_eos=True))
    assert asked == [2, "made"]
    assert {r.id: len(r.generated) for r in run_all(s)} == {a: 3, b: 3, c: 3}


def bare_llm(scheduler):
    """``LLM.generate`` over a scheduler without a device."""
    from tesseract_b200 import LLM

    llm = LLM.__new__(LLM)
    llm.scheduler, llm.config, llm.tokenizer = scheduler, scheduler.config, None
    llm._check_device_waits = lambda: None
    return llm


@pytest.mark.parametrize("refused, error", [
    (dict(allowed_token_ids=[2000]), ValueError), (dict(logit_bias={2001: 1.0}), ValueError), (dict(max_tokens=5000), RequestRejected),
    (dict(presence_penalty=1.0), RequestRejected)], ids=str)
def test_a_request_that_is_refused_leaves_nothing_of_its_call_behind(refused, error):
    """The call raises before any of its requests is taken, however many wait, and the next one runs."""
    s, fake = make()

    def no_room():
        raise MemoryError("nothing left on the device")

    s.prepare_rules = no_room
    llm = bare_llm(s)
    same = dict(max_tokens=3, temperature=0.0, ignore_eos=True)
    plain, prompts = SamplingParams(**same), [[k + 1] for k in range(20)]       # (more than fit at once)
    for place in (1, 19):
        with pytest.raises(error):
            llm.generate(prompts, [SamplingParams(**{**same, **refused}) if k == place else plain for k in range(20)])
        assert not s.has_work() and not s.requests and fake.batches == []
    with pytest.raises(RequestRejected):
        llm.generate([[1], []], plain)
    assert not s.has_work()
    assert [o.token_ids for o in llm.generate(prompts, plain)] == [[1000, 1001, 1002]] * 20
    fake.cache.check()
