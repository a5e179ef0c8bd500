"""Beam search, scoring and continuations on the engine, against the plain model and against requests of their own."""

import itertools
import json
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from tests.helpers import REL, TINY, random_tokens
from tests.plain import llama

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def log_softmax(x):
    x = np.asarray(x, dtype=np.float64)
    m = x.max(axis=-1, keepdims=True)
    return x - m - np.log(np.exp(x - m).sum(axis=-1, keepdims=True))


def plain_search(config, tensors, prompt, width, steps):
    """Every beam's whole sequence through the plain model each step; also the smallest margin of a choice."""
    beams, margin = [([], 0.0)], math.inf
    for _ in range(steps):
        every = []
        for place, (tokens, total) in enumerate(beams):
            logs = log_softmax(llama.forward(config, tensors, prompt + tokens)[-1].numpy())
            order = np.argsort(-logs, kind="stable")[:2 * width]
            every += [(-(total + logs[t]), place, rank, int(t)) for rank, t in enumerate(order)]
        every.sort()
        margin = min(margin, every[width][0] - every[width - 1][0])
        beams = [(beams[place][0] + [token], -negative) for negative, place, _, token in every[:width]]
    return beams, margin


def engine(folder, dtype="float32", **options):
    from tesseract_b200 import LLM

    options = {**dict(kv_capacity_tokens=2048, max_running=16, prefill_chunk_tokens=32, max_batch_tokens=96), **options}
    return LLM(folder, dtype=dtype, **options)


@pytest.mark.parametrize("share", [True, False])
@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("name, length, width, steps", [("a", 9, 4, 7), ("b", 65, 3, 8), ("c", 130, 8, 6), ("c", 300, 5, 4)])
def test_beams_in_32_bits_are_the_plain_searchs(model_folders, monkeypatch, name, length, width, steps, graphs, share):
    from tesseract_b200 import plan

    monkeypatch.setattr(plan, "SHARED_MIN_SAVED", 0)
    monkeypatch.setattr(plan, "SHARED_MIN_BYTES", 0 if share else 1 << 60)
    folder = model_folders(name)
    config, tensors = llama.load_folder(folder)
    prompts = [random_tokens(config["vocab_size"], length, seed=length), random_tokens(config["vocab_size"], length // 2, seed=1)]
    llm = engine(folder, cuda_graphs=graphs)
    found = llm.beam_search(prompts, width, steps, ignore_eos=True)
    for prompt, outs in zip(prompts, found):
        beams, margin = plain_search(config, tensors, prompt, width, steps)
        assert len(outs) == width and all(o.finish_reason == "length" and len(o.token_ids) == steps for o in outs)
        if margin > 1e-4:                              # (32-bit logits of these models are off by less than a tenth of that)
            assert sorted(o.token_ids for o in outs) == sorted(tokens for tokens, _ in beams)
        for out in outs:
            logs = log_softmax(llama.forward(config, tensors, prompt + out.token_ids).numpy())
            want = [logs[len(prompt) + k - 1, token] for k, token in enumerate(out.token_ids)]
            assert np.abs(np.asarray(out.token_logprobs) - want).max() < 1e-4
            assert out.score == pytest.approx(sum(out.token_logprobs), abs=1e-6)
        assert [o.score for o in outs] == sorted((o.score for o in outs), reverse=True)
    assert llm.stepper.cache.used_pages() == 0
    llm.stepper.cache.check()
    if graphs:
        assert bool(llm.stepper.graphs.shared_graphs) == (share and length >= 64)      # (a whole block in common)


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("name", ["a", "b", "c"])
def test_beams_in_bfloat16_are_scored_as_the_plain_model_scores_them(model_folders, monkeypatch, name, graphs):
    from tesseract_b200 import plan

    monkeypatch.setattr(plan, "SHARED_MIN_SAVED", 0)
    monkeypatch.setattr(plan, "SHARED_MIN_BYTES", 0)
    folder = model_folders(name)
    config, tensors = llama.load_folder(folder)
    length = 100
    prompts = [random_tokens(config["vocab_size"], length, seed=3)]
    llm = engine(folder, "bfloat16", cuda_graphs=graphs)
    for out in llm.beam_search(prompts, 6, 12, ignore_eos=True)[0]:
        logits = llama.forward(config, tensors, prompts[0] + out.token_ids).numpy()
        logs = log_softmax(logits)
        want = [logs[length + k - 1, token] for k, token in enumerate(out.token_ids)]
        # a log probability is a logit less the logarithm of a sum of them: each off by the engine's bound on a logit
        assert np.abs(np.asarray(out.token_logprobs) - want).max() <= 2 * REL["bfloat16"] * np.abs(logits).max()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_graphs_of_many_groupings(model_folders, monkeypatch, dtype):
    """Steps whose rows are grouped in many ways, more than there are graphs of exact sizes, against steps of twins launch by launch
    that share nothing."""
    from tesseract_b200 import plan
    from tesseract_b200.engine import StepEntry
    from tesseract_b200.engine.graph import GROUPINGS

    monkeypatch.setattr(plan, "SHARED_MIN_SAVED", 0)
    llm = engine(model_folders("b"), dtype, kv_capacity_tokens=16384, max_running=40)
    stepper, cache = llm.stepper, llm.stepper.cache
    prompts = {"p": random_tokens(384, 130, seed=1), "q": random_tokens(384, 200, seed=2)}
    for twin in "ab":
        for name, prompt in prompts.items():
            assert cache.admit((twin, name, 0), reserve_tokens=260)
            for k in range(0, len(prompt), 32):
                stepper.step([StepEntry((twin, name, 0), prompt[k:k + 32], [])])
            assert cache.fork([((twin, name, 0), (twin, name, k)) for k in range(1, 8)], reserve_tokens=260)
    sizes = [(8, 8), (7, 8), (6, 8), (5, 8), (4, 8), (3, 8), (2, 8), (8, 5), (8, 1), (7, 7), (6, 5), (8, 4), (8, 8), (3, 6), (5, 5), (8, 2)]
    for step, (first, second) in enumerate(sizes):
        rows = [("p", k) for k in range(first)] + [("q", k) for k in range(second)]
        tokens = random_tokens(384, len(rows), seed=step)
        entries = {twin: [StepEntry((twin, *row), [token], [0]) for row, token in zip(rows, tokens)] for twin in "ab"}
        monkeypatch.setattr(plan, "SHARED_MIN_BYTES", 0)
        launch = stepper.graphs.launch(entries["a"], [0.0] * len(rows), [0.0] * len(rows))
        got = launch.graph.logits[:launch.count].clone()
        monkeypatch.setattr(plan, "SHARED_MIN_BYTES", 1 << 60)
        want = stepper.step(entries["b"])
        assert float((got - want).abs().max()) <= REL[dtype] * float(want.abs().max())
    keys = list(stepper.graphs.shared_graphs)
    assert sum(1 for key in keys if key[0] == 16 and isinstance(key[2], tuple)) == GROUPINGS
    assert any(isinstance(key[2], int) for key in keys)


def test_one_beam_is_greedy_generation(model_folders):
    from tesseract_b200 import SamplingParams

    folder = model_folders("b")
    llm = engine(folder)
    prompts = [random_tokens(384, n, seed=n) for n in (5, 40, 70)]
    greedy = llm.generate(prompts, SamplingParams(max_tokens=10, temperature=0.0, ignore_eos=True))
    beams = llm.beam_search(prompts, 1, 10, ignore_eos=True)
    assert [outs[0].token_ids for outs in beams] == [out.token_ids for out in greedy]
    again = llm.generate(prompts, SamplingParams(max_tokens=10, temperature=0.0, ignore_eos=True))
    assert [out.token_ids for out in again] == [out.token_ids for out in greedy]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 64, 65, 100])
def test_scores_are_the_plain_models(model_folders, length, dtype):
    folder = model_folders("a")
    config, tensors = llama.load_folder(folder)
    sequence = random_tokens(config["vocab_size"], length, seed=length)
    llm = engine(folder, dtype)
    got = llm.score([sequence], alternatives=5)[0]
    assert got.token_ids == sequence and len(got.logprobs) == len(got.entropies) == len(got.alternatives) == length - 1
    if length > 1:
        logits = llama.forward(config, tensors, sequence).numpy()[:-1]
        logs = log_softmax(logits)
        bound = 2 * REL[dtype] * np.abs(logits).max() + 1e-5
        assert np.abs(np.asarray(got.logprobs) - logs[np.arange(length - 1), sequence[1:]]).max() <= bound
        # the entropy's derivative by a logit is p (ln p + H): its sum over the vocabulary is at most H + ln V
        entropy = -(np.exp(logs) * logs).sum(axis=1)
        assert np.abs(np.asarray(got.entropies) - entropy).max() <= bound * 2 * math.log(config["vocab_size"])
        best = np.sort(logs, axis=1)[:, ::-1][:, :5]
        assert np.abs(np.asarray([[v for _, v in row] for row in got.alternatives]) - best).max() <= bound
        assert got.perplexity == pytest.approx(math.exp(-np.mean(got.logprobs)))
    assert llm.stepper.cache.used_pages() == 0


def test_an_engine_at_work_refuses(model_folders):
    from tesseract_b200 import SamplingParams

    llm = engine(model_folders("a"))
    llm.scheduler.add_request([1, 2, 3], SamplingParams(max_tokens=4))
    for call in (lambda: llm.beam_search([[1]], 2, 3), lambda: llm.score([[1, 2]])):
        with pytest.raises(RuntimeError, match="idle"):
            call()


def designs():
    from tests.kazodra_models import TINY_KAZODRA
    from tests.ladedra_models import TINY_LADEDRA
    from tests.pekodra_models import TINY_PEKODRA
    from tests.revesun_models import TINY_REVESUN
    from tests.rirulix_models import TINY_RIRULIX
    from tests.tibivik_models import TINY_TIBIVIK

    made = {"llama": TINY["b"]}
    for name, models in (("revesun", TINY_REVESUN), ("pekodra", TINY_PEKODRA), ("kazodra", TINY_KAZODRA), ("ladedra", TINY_LADEDRA),
                         ("rirulix", TINY_RIRULIX), ("tibivik", TINY_TIBIVIK)):
        made[name] = next(iter(models.values()))
    return made


@pytest.mark.parametrize("design", ["llama", "revesun", "pekodra", "kazodra", "ladedra", "rirulix", "tibivik"])
@pytest.mark.parametrize("length", [3, 16, 37])
def test_a_continuation_goes_on_as_a_request_of_its_own_would(tmp_path, design, length):
    """Every design's caches and states fork: the same steps with two forked requests and with two that ran the whole prompt
    give the same logits, bit for bit in 32 bits."""
    from tesseract_b200.engine import StepEntry, load_model, make_stepper
    from tesseract_b200.weights.random_init import write_random_model

    config = dict(designs()[design])
    vocab = config.get("vocab_size") or config["vocab"]
    folder = write_random_model(str(tmp_path), dict(config, torch_dtype="float32"), 3)
    stepper = make_stepper(load_model(folder, dtype="float32"), capacity_tokens=512, max_requests=6, max_step_tokens=64)
    cache = stepper.cache
    prompt = [t % vocab for t in random_tokens(vocab, length, seed=length)]
    tails = [[t % vocab for t in random_tokens(vocab, 20, seed=s)] for s in (1, 2, 3)]

    def steps(requests):
        out = []
        for k in range(0, 18):
            out.append(stepper.step([StepEntry(r, [tail[k]], [0]) for r, tail in zip(requests, tails)]).cpu())
        out.append(stepper.step([StepEntry(r, tail[18:], [0, 1]) for r, tail in zip(requests, tails)]).cpu())
        return out

    for r in "xyz":
        assert cache.admit(r, reserve_tokens=100)
        stepper.step([StepEntry(r, prompt, [])])
    want = steps("xyz")
    for r in "xyz":
        cache.release(r)
    assert cache.admit("p", reserve_tokens=100)
    stepper.step([StepEntry("p", prompt, [])])
    assert cache.fork([("p", "q"), ("p", "s")], reserve_tokens=100)
    got = steps("pqs")
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    cache.release("p")
    cache.compact()                                    # what is left moves to the front, and goes on
    cache.check()
    left = stepper.step([StepEntry(r, [tail[0]], [0]) for r, tail in zip("qs", tails)]).cpu()
    for r, tail in zip("tu", tails[1:]):
        assert cache.admit(r, reserve_tokens=100)
        stepper.step([StepEntry(r, prompt, [])])
        for k in range(18):
            stepper.step([StepEntry(r, [tail[k]], [])])
        stepper.step([StepEntry(r, tail[18:], [])])
    fresh = stepper.step([StepEntry(r, [tail[0]], [0]) for r, tail in zip("tu", tails)]).cpu()
    assert float((left - fresh).abs().max()) <= REL["float32"] * float(fresh.abs().max())
    for r in "qstu":
        cache.release(r)
    assert cache.used_pages() == 0
    cache.check()


def test_the_command_line_scores_and_searches(model_folders):
    def run(*flags):
        done = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "tesseract"), "--model-path", model_folders("a"),
                               "--prompt-ids", "1,2,3,4", "--json", "--dtype", "float32", "--kv-capacity-tokens", "512", *flags],
                              capture_output=True, text=True, timeout=600)
        assert done.returncode == 0, done.stderr
        return [json.loads(line) for line in done.stdout.splitlines()]

    beams = run("--beams", "3", "--max-tokens", "4", "--ignore-eos")
    assert [b["beam"] for b in beams] == [0, 1, 2] and all(len(b["token_ids"]) == 4 for b in beams)
    (scored,) = run("--score")
    assert len(scored["logprobs"]) == 3 and scored["perplexity"] > 1.0


@pytest.mark.parametrize("width, ends", [(2, range(3, 13)), (4, range(0, 380)), (4, range(0, 200)), (32, range(0, 320, 3))])
def test_ids_that_end_a_beam_beyond_those_one_call_ranks(model_folders, width, ends):
    """Up to more ends than a ranking holds: what goes on and what ends is what the ranking of the whole vocabulary says."""
    folder, steps, ends = model_folders("b"), 4, set(ends)
    config, tensors = llama.load_folder(folder)
    prompt = random_tokens(config["vocab_size"], 20, seed=width)
    outs = engine(folder, max_running=40).beam_search([prompt], width, steps, stop_token_ids=sorted(ends), ignore_eos=True)[0]
    beams, finished, margin = [([], 0.0)], [], math.inf
    while beams and len(finished) < width and len(beams[0][0]) < steps:
        every = []
        for tokens, total in beams:
            logs = log_softmax(llama.forward(config, tensors, prompt + tokens)[-1].numpy())
            every += [(-(total + logs[t]), tokens + [t]) for t in range(config["vocab_size"])]
        every.sort()
        going = [(tokens, -negative) for negative, tokens in every if tokens[-1] not in ends]
        margin = min([margin, every[width][0] - every[width - 1][0]] + [a[1] - b[1] for a, b in zip(going[width - 1:], going[width:])][:1])
        finished += [(tokens, -negative) for negative, tokens in every[:width] if tokens[-1] in ends]
        beams = going[:width]
    if beams and len(beams[0][0]) >= steps:
        finished += beams
    want = sorted(finished, key=lambda f: -f[1])
    margin = min([margin] + [a[1] - b[1] for a, b in zip(want, want[1:width + 1])])
    for out in outs:
        logs = log_softmax(llama.forward(config, tensors, prompt + out.token_ids).numpy())
        scored = [logs[len(prompt) + k - 1, token] for k, token in enumerate(out.token_ids)]
        assert np.abs(np.asarray(out.token_logprobs) - scored).max() < 1e-4
    assert len(outs) == min(width, len(want))
    if margin > 1e-4:                                  # (32-bit logits of these models are off by less than a tenth of that)
        assert [out.token_ids for out in outs] == [tokens for tokens, _ in want[:width]]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_captured_step_whose_rows_grow(tmp_path, monkeypatch, dtype):
    """A group captured right behind its fork whose rows' own keys grow to many blocks: the same graph, against steps of twins launch
    by launch that share nothing."""
    from tesseract_b200 import plan
    from tesseract_b200.engine import StepEntry

    from tesseract_b200.weights.random_init import write_random_model

    monkeypatch.setattr(plan, "SHARED_MIN_SAVED", 0)
    folder = write_random_model(str(tmp_path), dict(TINY["b"], max_position_embeddings=4096, torch_dtype="float32"), 3)
    llm = engine(folder, dtype, kv_capacity_tokens=32768)
    stepper, cache = llm.stepper, llm.stepper.cache
    prompt = random_tokens(384, 1090, seed=1)
    for twin in "ab":
        assert cache.admit((twin, 0), reserve_tokens=2040)
        for k in range(0, len(prompt), 64):
            stepper.step([StepEntry((twin, 0), prompt[k:k + 64], [])])
        assert cache.fork([((twin, 0), (twin, k)) for k in range(1, 4)], reserve_tokens=2040)
    for own in (0, 1, 60, 130, 300, 700, 940):
        for k in range(4):                             # (a portion a row, up to the next step that is compared; row 3 stays behind)
            grown = own - (cache.length(("a", k)) - len(prompt)) if k < 3 else 0
            tokens = random_tokens(384, max(1, grown), seed=own + k)
            for twin in "ab":
                for at in range(0, grown, 64):
                    stepper.step([StepEntry((twin, k), tokens[at:min(at + 64, grown)], [])])
        tokens = random_tokens(384, 4, seed=own + 9)
        entries = {twin: [StepEntry((twin, k), [tokens[k]], [0]) for k in range(4)] for twin in "ab"}
        monkeypatch.setattr(plan, "SHARED_MIN_BYTES", 0)
        launch = stepper.graphs.launch(entries["a"], [0.0] * 4, [0.0] * 4)
        got = launch.graph.logits[:launch.count].clone()
        monkeypatch.setattr(plan, "SHARED_MIN_BYTES", 1 << 60)
        want = stepper.step(entries["b"])
        assert float((got - want).abs().max()) <= REL[dtype] * float(want.abs().max())
    (graph,) = stepper.graphs.shared_graphs.values()   # (one capture serves all)
    shared = next(view.shared for view in graph.ctx.groups if view.shared is not None)
    (choice,) = shared.plans.values()
    assert choice.tail_parts > 4 and choice.prefix_parts > 4


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_rule_itself_sends_a_step_to_keys_in_common(tmp_path, monkeypatch, dtype):
    """With the thresholds as they are: 32 continuations of a long prompt take the path that reads common keys once, in a graph and launch
    by launch, few do not; results are those of steps that share nothing."""
    from tesseract_b200 import plan
    from tesseract_b200.engine import StepEntry
    from tesseract_b200.weights.random_init import write_random_model

    config = dict(TINY["b"], num_key_value_heads=3, max_position_embeddings=8192, torch_dtype="float32")
    llm = engine(write_random_model(str(tmp_path), config, 3), dtype, kv_capacity_tokens=16384, max_running=72, max_batch_tokens=512,
                 prefill_chunk_tokens=512)
    stepper, cache = llm.stepper, llm.stepper.cache
    rows, prompt = 32, random_tokens(384, 64 * plan.SHARED_LONG + 70, seed=1)
    saved = (rows - 1) * (len(prompt) // 64) * cache.shared_block_bytes
    assert plan.SHARED_MIN_BYTES // 3 <= saved < 4 * plan.SHARED_MIN_BYTES
    for twin in "ab":
        assert cache.admit((twin, 0), reserve_tokens=len(prompt) + 20)
        for k in range(0, len(prompt), 512):
            stepper.step([StepEntry((twin, 0), prompt[k:k + 512], [])])
        assert cache.fork([((twin, 0), (twin, k)) for k in range(1, rows)], reserve_tokens=len(prompt) + 20)

    def entries(twin, count, seed):
        return [StepEntry((twin, k), [token], [0]) for k, token in enumerate(random_tokens(384, count, seed=seed))]

    def alike(got, want):
        return float((got - want).abs().max()) <= REL[dtype] * float(want.abs().max())

    least = plan.SHARED_MIN_BYTES
    few = 1 + least // 4 // (len(prompt) // 64 * cache.shared_block_bytes)           # (saves less than a third of the threshold)
    for step, (count, shares) in enumerate([(rows, True), (few, False), (rows, True)]):
        assert (stepper.company(entries("a", count, step)) is not None) == shares
        made = len(stepper.graphs.shared_graphs)
        if step < 2:
            launch = stepper.graphs.launch(entries("a", count, step), [0.0] * count, [0.0] * count)
            got = launch.graph.logits[:count].clone()
            assert (len(stepper.graphs.shared_graphs) > made) == shares
        else:
            got = stepper.step(entries("a", count, step)).clone()
        monkeypatch.setattr(plan, "SHARED_MIN_BYTES", 1 << 60)
        want = stepper.step(entries("b", count, step))
        monkeypatch.setattr(plan, "SHARED_MIN_BYTES", least)
        assert alike(got, want)
