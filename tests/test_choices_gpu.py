"""Requests that say something about their next tokens, through the engine: against the plain model under the same rules, alone and
beside others, with and without captured steps."""

import json
import math
import os
import subprocess
import sys

import numpy as np
import pytest

from tests import token_choice_plain as plain
from tests.helpers import random_tokens
from tests.plain import llama
from tests.test_beam_gpu import log_softmax
from tests.test_generate_gpu import plain_next

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def engine(folder, dtype="float32", **options):
    from tesseract_b200 import LLM

    return LLM(folder, dtype=dtype, **{**dict(kv_capacity_tokens=2048, max_running=8, prefill_chunk_tokens=32, max_batch_tokens=96),
                                       **options})


def ruled_logits(logits, params, prompt, generated, allowed=None):
    vocab = logits.size
    seen, counts = np.zeros(vocab, dtype=bool), np.zeros(vocab, dtype=np.int64)
    seen[list(prompt) + list(generated)] = True
    np.add.at(counts, np.asarray(generated, dtype=np.int64), 1)
    rule = (params.repetition_penalty, params.presence_penalty, params.frequency_penalty) if params.penalised else None
    mask = None
    for ids in (params.allowed_token_ids, allowed):
        if ids is not None:
            mine = np.zeros(vocab, dtype=bool)
            mine[list(ids)] = True
            mask = mine if mask is None else mask & mine
    return plain.shaped(logits, rule, seen, counts, params.logit_bias, mask)


def test_a_sampler_keeps_the_tokens_of_rows_beside_top_p():
    """Rows that top-p says nothing of have, beside one that it cuts, the token that they have without it, with NaN and +inf too; a row
    that it cuts with such logits is refused."""
    import torch

    from tesseract_b200.sampling.sampler import InvalidLogits, Sampler

    logits = np.random.RandomState(3).randn(6, 500).astype(np.float32)
    logits[1, 40] = np.inf
    logits[2, 3:9] = np.nan
    logits[3] = np.nan
    logits[4, 7] = np.inf
    sampler, on_device = Sampler("cuda"), torch.from_numpy(logits).cuda()
    temperatures, draws = [0.7, 0.0, 0.0, 0.0, 0.7, 0.7], [0.1, 0.2, 0.3, 0.4, 0.5, 0.6]
    alone = sampler.sample(on_device, temperatures, [1.0] * 6, draws)
    beside = sampler.sample(on_device, temperatures, [0.5] + [1.0] * 5, draws)
    assert beside[1:] == alone[1:]
    assert beside[0] == plain.choose(logits[0], 0.7, 0.1, 0, 0.5, 0.0)
    with pytest.raises(InvalidLogits):
        sampler.sample(on_device, temperatures, [1.0] * 4 + [0.5] * 2, draws)


def check_answer(config, tensors, prompt, params, out):
    """Every token is the plain model's under the rules; 32-bit logits may be off by 1e-5 of the largest, so a greedy token may be that
    much below the best, and a drawn one that of a draw (or of a temperature) a little beside it."""
    rng, tokens = llama.SplitMix64(params.seed) if params.temperature > 0 else None, []
    for got in out:
        logits = plain_next(config, tensors, list(prompt) + tokens)
        x = ruled_logits(logits, params, prompt, tokens, params.grammar(tuple(tokens)) if params.grammar else None)
        assert x[got] > -np.inf
        if rng is None:
            assert x.max() - x[got] <= 1e-5 * np.abs(logits).max()
        else:
            draw = rng.unit_f64()
            near = {plain.choose(x.astype(np.float32), params.temperature * t, min(max(draw + e, 0.0), 1 - 1e-9), params.top_k, params.top_p,
                                 params.min_p) for e in (0.0, 1e-4, -1e-4) for t in (1.0, 1 + 1e-4, 1 - 1e-4)}
            assert got in near
        tokens.append(int(got))


def many_kinds(vocab):
    from tesseract_b200 import SamplingParams

    def even_then_odd(tokens):
        return range(len(tokens) % 2, vocab, 2)

    def counting(tokens):                                    # one token may follow, then some
        return [7] if not tokens or tokens[-1] != 7 else [7, 8, 9, 30, vocab - 1]

    same = dict(max_tokens=14, ignore_eos=True)
    return [
        SamplingParams(temperature=0.0, repetition_penalty=1.7, **same),
        SamplingParams(temperature=0.0, presence_penalty=0.6, frequency_penalty=0.4, **same),
        SamplingParams(temperature=0.0, frequency_penalty=-0.3, logit_bias={5: 2.0, 9: -math.inf, vocab - 1: 1.0}, **same),
        SamplingParams(temperature=0.0, allowed_token_ids=[3, 4, 50, 60, vocab - 1], repetition_penalty=1.5, **same),
        SamplingParams(temperature=0.0, grammar=even_then_odd, presence_penalty=0.5, **same),
        SamplingParams(temperature=0.9, seed=31, top_p=0.8, **same),
        SamplingParams(temperature=1.2, seed=32, top_k=12, repetition_penalty=1.3, **same),
        SamplingParams(temperature=0.8, seed=33, min_p=0.05, logit_bias={t: 0.5 for t in range(40)}, **same),
        SamplingParams(temperature=1.0, seed=34, grammar=counting, **same),
        SamplingParams(temperature=1.0, seed=35, top_k=30, top_p=0.9, min_p=0.01, presence_penalty=0.4, **same),
        SamplingParams(temperature=0.7, seed=36, **same),                    # (and two that say nothing)
        SamplingParams(temperature=0.0, **same),
    ]


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("name", ["a", "b", "c"])
def test_answers_are_the_plain_models_under_the_rules(model_folders, name, graphs):
    folder = model_folders(name)
    config, tensors = llama.load_folder(folder)
    kinds = many_kinds(config["vocab_size"])
    prompts = [random_tokens(config["vocab_size"], 1 + (17 * k) % 70, seed=200 + k) for k in range(len(kinds))]
    llm = engine(folder, cuda_graphs=graphs)
    outs = llm.generate(prompts, kinds)
    for prompt, params, out in zip(prompts, kinds, outs):
        assert out.finish_reason == "length" and len(out.token_ids) == 14, out.error
        check_answer(config, tensors, prompt, params, out.token_ids)
    assert llm.stepper.cache.used_pages() == 0
    llm.stepper.cache.check()


def test_an_answer_does_not_depend_on_what_shares_its_batches(model_folders):
    """Alone in captured steps, and beside others through few slots, in small portions, with every step run launch by launch: slots with
    other requests' rules and histories behind them."""
    folder = model_folders("b")
    config, _ = llama.load_folder(folder)
    kinds = many_kinds(config["vocab_size"]) * 2
    prompts = [random_tokens(config["vocab_size"], 1 + (23 * k) % 60, seed=300 + k) for k in range(len(kinds))]
    alone = engine(folder, max_running=1)
    want = [alone.generate([prompt], params)[0].token_ids for prompt, params in zip(prompts, kinds)]
    for options in (dict(max_running=3, prefill_chunk_tokens=16, cuda_graphs=False), dict(max_running=5), dict(max_running=16)):
        llm = engine(folder, **options)
        assert [o.token_ids for o in llm.generate(prompts, kinds)] == want, options


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_steps_under_rules_and_cuts_are_launched_ahead(model_folders, dtype):
    """Captured steps note the tokens that they are fed on the device; the host reads them a step later."""
    from tesseract_b200 import SamplingParams

    folder = model_folders("b")
    config, _ = llama.load_folder(folder)
    prompts = [random_tokens(config["vocab_size"], n, seed=n) for n in (5, 30, 1)]
    same = dict(max_tokens=30, ignore_eos=True)
    for kinds in ([SamplingParams(temperature=0.0, repetition_penalty=1.4, frequency_penalty=0.2, **same)] * 3,
                  [SamplingParams(temperature=0.9, top_p=0.7, seed=9, **same)] * 3,
                  [SamplingParams(temperature=0.9, top_k=9, seed=9, **same), SamplingParams(temperature=0.0, logit_bias={3: 1.0}, **same),
                   SamplingParams(temperature=0.5, seed=4, **same)]):
        llm = engine(folder, dtype=dtype)
        launched = []
        launch = llm.stepper.launch_decode
        llm.scheduler.launch_decode = lambda *a: launched.append(len(a[0])) or launch(*a)
        got = [o.token_ids for o in llm.generate(prompts, kinds)]
        assert len(launched) >= 25
        if dtype == "float32":
            ordinary = engine(folder, dtype=dtype, cuda_graphs=False)
            assert got == [o.token_ids for o in ordinary.generate(prompts, kinds)]
        assert all(len(tokens) == 30 for tokens in got)


def test_penalties_keep_a_greedy_answer_from_repeating(model_folders):
    from tesseract_b200 import SamplingParams

    folder = model_folders("a")
    config, _ = llama.load_folder(folder)
    prompt = random_tokens(config["vocab_size"], 9, seed=1)
    llm = engine(folder)
    out = llm.generate([prompt], SamplingParams(max_tokens=100, temperature=0.0, presence_penalty=1e4, ignore_eos=True))[0]
    assert len(set(out.token_ids)) == 100                    # (each of 256 tokens at most once)


def test_a_request_that_allows_no_token_ends_alone(model_folders):
    from tesseract_b200 import SamplingParams

    folder = model_folders("b")
    config, tensors = llama.load_folder(folder)
    prompts = [random_tokens(config["vocab_size"], n, seed=n) for n in (5, 30, 8)]
    same = dict(max_tokens=10, temperature=0.0, ignore_eos=True)
    kinds = [SamplingParams(allowed_token_ids=[3], logit_bias={3: -math.inf}, **same), SamplingParams(repetition_penalty=1.2, **same),
             SamplingParams(grammar=lambda tokens: [] if len(tokens) == 4 else [5, 6], **same)]
    for graphs in (True, False):
        llm = engine(folder, cuda_graphs=graphs)
        outs = llm.generate(prompts, kinds)
        assert outs[0].finish_reason == "error" and outs[0].token_ids == [] and "no token" in outs[0].error
        assert outs[2].finish_reason == "error" and len(outs[2].token_ids) == 4 and set(outs[2].token_ids) <= {5, 6}
        assert outs[1].finish_reason == "length"
        check_answer(config, tensors, prompts[1], kinds[1], outs[1].token_ids)
        assert llm.stepper.cache.used_pages() == 0


def plain_ruled_search(config, tensors, prompt, width, steps, params):
    beams, margin = [([], 0.0)], math.inf
    for _ in range(steps):
        every = []
        for place, (tokens, total) in enumerate(beams):
            logits = llama.forward(config, tensors, prompt + tokens)[-1].numpy()
            logs = log_softmax(ruled_logits(logits, params, prompt, tokens))
            order = np.argsort(-logs, kind="stable")[:2 * width]
            every += [(-(total + logs[t]), place, rank, int(t)) for rank, t in enumerate(order) if logs[t] > -math.inf]
        every.sort()
        if len(every) > width:
            margin = min(margin, every[width][0] - every[width - 1][0])
        beams = [(beams[place][0] + [token], -negative) for negative, place, _, token in every[:width]]
    return beams, margin


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("name, length, width, steps", [("a", 9, 4, 8), ("b", 65, 3, 9), ("c", 130, 6, 6)])
def test_beams_under_rules(model_folders, name, length, width, steps, graphs):
    """A forked beam has its parent's history."""
    from tesseract_b200 import SamplingParams

    folder = model_folders(name)
    config, tensors = llama.load_folder(folder)
    prompts = [random_tokens(config["vocab_size"], length, seed=length), random_tokens(config["vocab_size"], length // 2, seed=1)]
    llm = engine(folder, cuda_graphs=graphs, max_running=16)
    for params in (SamplingParams(repetition_penalty=1.6, frequency_penalty=0.5),
                   SamplingParams(presence_penalty=0.7, logit_bias={3: 2.0, 10: -math.inf}, allowed_token_ids=range(2, 90))):
        found = llm.beam_search(prompts, width, steps, ignore_eos=True, rules=params)
        for prompt, outs in zip(prompts, found):
            beams, margin = plain_ruled_search(config, tensors, prompt, width, steps, params)
            assert len(outs) == width
            if margin > 1e-4:
                assert sorted(o.token_ids for o in outs) == sorted(tokens for tokens, _ in beams)
            for out in outs:
                for k, token in enumerate(out.token_ids):
                    logits = llama.forward(config, tensors, prompt + out.token_ids[:k])[-1].numpy()
                    want = log_softmax(ruled_logits(logits, params, prompt, out.token_ids[:k]))[token]
                    assert abs(out.token_logprobs[k] - want) < 1e-4
    assert llm.stepper.cache.used_pages() == 0


def test_beam_search_refuses_what_it_does_not_take(model_folders):
    from tesseract_b200 import SamplingParams

    llm = engine(model_folders("a"), cuda_graphs=False)
    for rules in (SamplingParams(grammar=lambda tokens: [1]), SamplingParams(logit_bias={256: 1.0}), SamplingParams(allowed_token_ids=[999])):
        with pytest.raises(ValueError):
            llm.beam_search([[1, 2]], 2, 3, rules=rules)


def test_command_line_takes_rules(model_folders):
    folder = model_folders("a")
    cmd = [sys.executable, os.path.join(ROOT, "bin", "tesseract"), "--model-path", folder, "--prompt-ids", "5,6,7,8", "--max-tokens", "6",
           "--temperature", "0", "--ignore-eos", "--json", "--kv-capacity-tokens", "256", "--max-running", "4", "--dtype", "float32",
           "--allowed-token-ids", "20,21,22,23,24,25,26", "--presence-penalty", "1000", "--logit-bias", "20:-inf"]
    for more, count in (([], 1), (["--beams", "2"], 2)):
        done = subprocess.run(cmd + more, capture_output=True, text=True, timeout=300)
        assert done.returncode == 0, done.stderr
        records = [json.loads(line) for line in done.stdout.strip().splitlines()]
        assert len(records) == count
        for record in records:
            assert sorted(record["token_ids"]) == [21, 22, 23, 24, 25, 26]
