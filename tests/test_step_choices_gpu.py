"""How the engine's steps choose their rows' tokens, captured and launched one by one, against the plain model."""

import decimal

import numpy as np
import pytest
import torch

from tesseract_b200 import kernels
from tests import token_choice_plain as choices
from tests.helpers import TINY, make_model_folder, random_tokens
from tests.plain import llama
from tests.test_choices_gpu import check_answer, engine

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [262144, 262145])
@pytest.mark.parametrize("graphs", [False, True])
def test_top_p_on_either_side_of_the_kernels_largest_vocabulary(tmp_path, vocab, graphs):
    """A row that top-p cuts beside a greedy one and one that is drawn from all (logits of some 0.11 from token to token: low temperatures,
    so that no draw falls among tokens that weigh a millionth each)."""
    from tesseract_b200 import SamplingParams

    folder = make_model_folder(str(tmp_path), {**TINY["a"], "num_hidden_layers": 1, "hidden_size": 32, "intermediate_size": 64,
                                               "vocab_size": vocab}, "bfloat16", 3)
    config, tensors = llama.load_folder(folder)
    same = dict(max_tokens=4, ignore_eos=True)
    kinds = [SamplingParams(temperature=0.03, top_p=0.15, seed=8, **same), SamplingParams(temperature=0.0, **same),
             SamplingParams(temperature=0.02, seed=7, **same)]
    prompts = [random_tokens(vocab, n, seed=n) for n in (41, 3, 40)]
    outs = engine(folder, cuda_graphs=graphs).generate(prompts, kinds)
    for prompt, params, out in zip(prompts, kinds, outs):
        assert out.finish_reason == "length" and len(out.token_ids) == 4, out.error
        check_answer(config, tensors, prompt, params, out.token_ids)


@pytest.mark.parametrize("rows", [6, 30, 200])
@pytest.mark.parametrize("vocab", [1, 3, 1000, 5000, 20000, 128256, 200000])
def test_logits_that_are_not_finite_give_a_marked_row_the_samplers_token(rows, vocab):
    """Equal tokens, with no tolerance: the row of ``sample`` in a call of as many rows.  Others have none."""
    rng = np.random.RandomState(rows + vocab)
    x = (rng.randn(rows, vocab) * 2).astype(np.float32)
    for row in range(rows):
        kind, some = row % 6, rng.permutation(vocab)[:1 + row % 3]
        if kind == 1:
            x[row, some] = np.nan
        elif kind == 2:
            x[row, some] = np.inf
        elif kind == 3:
            x[row] = np.nan if row % 4 < 2 else -np.inf
        elif kind == 4:
            x[row, vocab // 2:] = np.nan if row % 4 < 2 else -np.inf
            x[row, some] = np.nan
        elif kind == 5:
            x[row, some[0]], x[row, some[-1]] = np.inf, np.nan
    logits = torch.from_numpy(x).cuda()
    draws = torch.from_numpy(rng.rand(rows)).cuda()
    marked = torch.from_numpy((rng.rand(rows) < 0.7).astype(np.int32)).cuda()
    invalid = ~(x < np.inf).all(axis=1) | (x.max(axis=1) == -np.inf)
    for temperature in (0.0, 0.7, 1e-38, None):
        of_rows = np.full(rows, temperature) if temperature is not None else rng.choice([0.0, 0.4, 1.0, 2.0], rows)
        of_rows = torch.from_numpy(of_rows.astype(np.float32)).cuda()
        want, got = (torch.full((rows,), -9, dtype=torch.int32, device="cuda") for _ in range(2))
        kernels.sample(logits, of_rows, draws, want)
        kernels.choose_tokens(logits, of_rows, draws, got, as_sampled=marked)
        keep = marked.cpu().numpy() != 0
        want, got = want.cpu().numpy(), got.cpu().numpy()
        assert np.array_equal(got[invalid & keep], want[invalid & keep])
        assert (got[invalid & ~keep] == -1).all()
        if temperature != 1e-38:                 # (there the largest logit's own distance is rounded otherwise)
            assert np.array_equal(got[~invalid], want[~invalid])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("spoiled", ["nan", "inf", "all"])
def test_a_request_that_says_nothing_does_not_fail_for_its_neighbours_rules(model_folders, spoiled, graphs, dtype):
    """A model some of whose logits are not finite: a greedy request and one that is drawn from everything have the tokens beside
    requests with rules and cuts that they have beside each other."""
    from tesseract_b200 import SamplingParams

    llm = engine(model_folders("b"), dtype=dtype, cuda_graphs=graphs)
    weight = llm.model.head.proj.weight
    if spoiled == "all":
        weight.fill_(float("nan"))
    else:
        weight[7, 5] = float(spoiled)
    same = dict(max_tokens=8, ignore_eos=True)
    plain = [SamplingParams(temperature=0.0, **same), SamplingParams(temperature=0.8, seed=3, **same)]
    prompts = [random_tokens(384, n, seed=n) for n in (9, 20, 3)]
    alone = llm.generate(prompts, plain + [plain[1]])
    assert [o.finish_reason for o in alone] == ["length"] * 3
    for other in (SamplingParams(temperature=0.8, top_p=0.5, **same), SamplingParams(temperature=0.0, presence_penalty=0.5, **same),
                  SamplingParams(temperature=0.9, top_k=5, logit_bias={7: -1.0}, **same)):
        beside = llm.generate(prompts, plain + [other])
        assert [o.finish_reason for o in beside[:2]] == ["length"] * 2, [o.error for o in beside]
        assert [o.token_ids for o in beside[:2]] == [o.token_ids for o in alone[:2]]


def test_a_replayed_portion_that_fails_leaves_histories_as_they_were(model_folders):
    """Steps with a prompt's portion and its end, captured: tried again after a failure in front of the launch, their tokens are in
    the history once."""
    from tesseract_b200 import SamplingParams
    from tesseract_b200.engine.step import StepEntry
    from tesseract_b200.sampling.params import TokenChoice

    stepper = engine(model_folders("b")).stepper
    prompt = random_tokens(384, 50, seed=1)
    choice = TokenChoice.of(SamplingParams(temperature=0.0, frequency_penalty=0.5), 45)      # (the last five count as an answer's)

    def feed(request):
        slot = stepper.cache.slot(request)
        for part, want in ((prompt[:32], []), (prompt[32:], [17])):
            stepper.step([StepEntry(request, part, want, choice)])
        return stepper.rules.counts[slot].cpu().numpy(), stepper.rules.seen[slot].cpu().numpy()

    assert stepper.cache.admit("first") and stepper.cache.admit("second")
    counts, seen = feed("first")
    assert np.array_equal(counts, np.bincount(prompt[45:], minlength=384)) and stepper.chunk_graphs.replays == 2

    class Failing:
        def __init__(self, graph):
            self.graph, self.failed = graph, False

        def replay(self):
            if not self.failed:
                self.failed = True
                raise RuntimeError("injected")
            self.graph.replay()

    for graph in stepper.chunk_graphs.graphs.values():
        graph.graph = Failing(graph.graph)
    slot = stepper.cache.slot("second")
    for part, want in ((prompt[:32], []), (prompt[32:], [17])):
        with pytest.raises(RuntimeError, match="injected"):
            stepper.step([StepEntry("second", part, want, choice)])
        stepper.step([StepEntry("second", part, want, choice)])
    assert np.array_equal(stepper.rules.counts[slot].cpu().numpy(), counts)
    assert np.array_equal(stepper.rules.seen[slot].cpu().numpy(), seen)


def test_rules_without_room_on_the_device_fail_no_step(model_folders, monkeypatch):
    from tesseract_b200 import SamplingParams
    from tesseract_b200.engine.scheduler import RequestRejected
    from tesseract_b200.sampling import rules

    def no_room(*args, **kwargs):
        raise torch.OutOfMemoryError("CUDA out of memory")

    llm = engine(model_folders("a"))
    same = dict(max_tokens=6, temperature=0.0, ignore_eos=True)
    want = llm.generate([[1, 2, 3]], SamplingParams(**same))[0].token_ids
    first = llm.scheduler.add_request([1, 2, 3], SamplingParams(**same))
    with monkeypatch.context() as patch:
        patch.setattr(rules, "TokenRules", no_room)
        with pytest.raises(RequestRejected, match="out of memory"):
            llm.scheduler.add_request([4], SamplingParams(presence_penalty=1.0, **same))
    second = llm.scheduler.add_request([4], SamplingParams(presence_penalty=1e4, **same))
    done = {}
    while llm.scheduler.has_work():
        done.update({r.id: r for r in llm.scheduler.step().finished})
    assert done[first].generated == want and len(set(done[second].generated)) == 6


def test_weights_are_those_of_64_bits():
    """Two tokens, draws and top-p on either side of the border between them.  A weight e^-d is off by: its series behind r^4, r^5 / 120
    with |r| <= ln 2 / 512, below 2^-54; the table's power of two, 2^-52; r's two roundings, d 2^-53 and less; four roundings on the way,
    2^-53 each: 2^-50 (1 + d / 2) holds them all.  The border w0 / (w0 + w1) moves by no more, and the sums, products and the draw itself
    are rounded by 2^-53 each, 2^-51 together."""
    rng = np.random.RandomState(5)
    d = rng.uniform(0.01, 4.0, 4000).astype(np.float32)
    x = np.full((d.size, 3), -1e30, dtype=np.float32)
    x[:, 0], x[:, 1] = 0.0, -d
    logits = torch.from_numpy(x).cuda()
    ones, out = torch.ones(d.size, device="cuda"), torch.empty(d.size, dtype=torch.int32, device="cuda")
    with decimal.localcontext(prec=40):
        border = [1 / (1 + (-decimal.Decimal(float(v))).exp()) for v in d]
        off = [decimal.Decimal(2.0 ** -50 * (1.0 + 0.5 * float(v)) + 2.0 ** -51) for v in d]
        sides = [np.array([float(b * (1 + sign * o)) for b, o in zip(border, off)]) for sign in (-1, 1)]
    for token, side in enumerate(sides):
        draws = torch.from_numpy(side).cuda()
        for cut in (None, torch.full((d.size,), 2, dtype=torch.int32, device="cuda")):       # (in the order of ids, and of the rank)
            kernels.choose_tokens(logits, ones, draws, out, top_k=cut)
            assert (out == token).all()
        late = torch.full((d.size,), 1.0 - 2.0 ** -20, dtype=torch.float64, device="cuda")
        kernels.choose_tokens(logits, ones, late, out, top_p=draws)                          # (the first alone is kept, or both)
        assert (out == token).all()


@pytest.mark.parametrize("vocab", [3, 100, 20000, 128256])
@pytest.mark.parametrize("below", [699.0, 701.0, 712.5, 730.0, 744.0, 745.0, 746.0, 800.0])
def test_a_draw_of_nothing_takes_the_samplers_first_token(vocab, below):
    """A row without a cut: the first token whose weight is a number of 64 bits above 0, down to e^-745.  (That is 5.0e-324, and the
    least number above 0 is 4.9e-324: a library's exp that is a unit off may give 0.  e^-744, 1.36e-323, is further from it.)"""
    x = np.full((3, vocab), -1e4, dtype=np.float32)
    x[:, -1] = 3.0
    x[1, vocab // 2] = x[2, 0] = 3.0 - below
    logits = torch.from_numpy(x).cuda()
    ones, draws = torch.ones(3, device="cuda"), torch.zeros(3, dtype=torch.float64, device="cuda")
    want, got = (torch.full((3,), -9, dtype=torch.int32, device="cuda") for _ in range(2))
    kernels.sample(logits, ones, draws, want)
    kernels.choose_tokens(logits, ones, draws, got)
    first = [vocab - 1, vocab // 2, 0] if below < 745.5 else [vocab - 1] * 3
    assert got.tolist() == want.tolist()
    assert first == [choices.choose(row, 1.0, 0.0) for row in x] and (got.tolist() == first or below == 745.0)


@pytest.mark.parametrize("temperature", [2e-3, 2e-4, 1e-4, 1e-5, 1e-6, 1e-8])
def test_a_marked_row_has_the_samplers_token_at_low_temperatures(temperature):
    """Logits a few units of their last place apart, whose distances from the largest are rounded in one way by ``sample`` and in another
    for cuts: a row without a cut has ``sample``'s tokens.  Each side sums in 64 bits, 2,000 weights, in its own order: 2^-42 of the whole
    at most, within which a draw falls once in 10^8 rows."""
    rng = np.random.RandomState(3)
    rows, vocab = 400, 2000
    steps = rng.randint(0, 40, (rows, vocab)).astype(np.float32)
    x = (np.float32(15.7) + steps * np.float32(2.0 ** -20)) * rng.choice([1.0, -1.0, 0.25], (rows, 1)).astype(np.float32)
    x = x.astype(np.float32)
    logits = torch.from_numpy(x).cuda()
    of_rows, draws = torch.full((rows,), temperature, device="cuda"), torch.from_numpy(rng.rand(rows)).cuda()
    want, got = (torch.full((rows,), -9, dtype=torch.int32, device="cuda") for _ in range(2))
    kernels.sample(logits, of_rows, draws, want)
    kernels.choose_tokens(logits, of_rows, draws, got, as_sampled=torch.ones(rows, dtype=torch.int32, device="cuda"))
    assert got.tolist() == want.tolist()
    # (a mark says nothing about a row with a cut)
    cut = torch.full((rows,), 0.9, dtype=torch.float64, device="cuda")
    without = kernels.choose_tokens(logits, of_rows, draws, want, top_p=cut).tolist()
    assert kernels.choose_tokens(logits, of_rows, draws, got, top_p=cut, as_sampled=torch.ones(rows, dtype=torch.int32, device="cuda")).tolist() == without


@pytest.mark.parametrize("rows, vocab", [(70, 131073), (30, 200001), (150, 262144)])
def test_more_rows_than_fit_at_once_of_more_than_eight_blocks(rows, vocab):
    rng = np.random.RandomState(rows)
    x = (rng.randn(rows, vocab) * 2.5).astype(np.float32)
    temperature, draws = rng.choice([0.0, 0.6, 1.0, 1.5], rows).astype(np.float32), rng.rand(rows)
    top_k, top_p = rng.choice([0, 0, 5, 3000], rows).astype(np.int32), rng.choice([1.0, 1.0, 0.9, 0.4], rows)
    out = torch.full((rows,), -9, dtype=torch.int32, device="cuda")
    kernels.choose_tokens(*(torch.from_numpy(a).cuda() for a in (x, temperature, draws)), out, top_k=torch.from_numpy(top_k).cuda(),
                          top_p=torch.from_numpy(top_p).cuda())
    assert out.tolist() == [choices.choose(x[r], temperature[r], draws[r], top_k[r], top_p[r]) for r in range(rows)]


def test_top_p_of_a_sampler_draws_from_what_is_not_ruled_out():
    """Logits of -inf weigh nothing; a row that top-p cuts of which NaN, +inf or nothing is left is refused."""
    from tesseract_b200.sampling.sampler import InvalidLogits, Sampler

    rng = np.random.RandomState(8)
    x = (rng.randn(4, 700) * 2).astype(np.float32)
    x[0, rng.permutation(700)[:600]] = -np.inf
    x[1, 1:] = -np.inf
    sampler, draws = Sampler("cuda"), [0.2, 0.9, 0.5, 0.7]
    got = sampler.sample(torch.from_numpy(x).cuda(), [0.9] * 4, [0.8, 0.5, 0.9, 1.0], draws)
    assert got == [choices.choose(x[r], 0.9, draws[r], 0, p) for r, p in enumerate((0.8, 0.5, 0.9, 1.0))]
    for spoiled in (np.full(700, -np.inf), np.where(np.arange(700) == 3, np.nan, x[2]), np.where(np.arange(700) == 3, np.inf, x[2])):
        x[2] = spoiled
        with pytest.raises(InvalidLogits):
            sampler.sample(torch.from_numpy(x).cuda(), [0.9] * 4, [0.8, 0.5, 0.9, 1.0], draws)


def test_kinds_of_captured_steps_follow_one_another(model_folders):
    """Requests with rules, cuts and neither that begin and end at different steps, so that a batch goes from one kind of captured step
    to another while rows are in flight: each has the answer that it has alone."""
    from tesseract_b200 import SamplingParams

    folder = model_folders("b")

    def kind(k, tokens):
        same = dict(max_tokens=tokens, ignore_eos=True, seed=k)
        return [SamplingParams(temperature=0.0, **same), SamplingParams(temperature=0.9, **same), SamplingParams(temperature=0.9, top_p=0.7, **same),
                SamplingParams(temperature=0.8, top_k=7, frequency_penalty=0.4, **same), SamplingParams(temperature=0.0, repetition_penalty=1.4, **same),
                SamplingParams(temperature=0.7, min_p=0.1, **same)][k % 6]

    # (and ten that say nothing at the end)
    kinds = [kind(k, 2 + (7 * k) % 23) for k in range(30)] + [kind(k % 2, 4 + k) for k in range(10)]
    prompts = [random_tokens(384, 1 + (5 * k) % 9, seed=400 + k) for k in range(40)]
    alone = engine(folder, max_running=1)
    want = [alone.generate([prompt], params)[0].token_ids for prompt, params in zip(prompts, kinds)]
    for running in (3, 5, 8):
        llm = engine(folder, max_running=running)
        assert [o.token_ids for o in llm.generate(prompts, kinds)] == want
        graphs = llm.stepper.graphs
        assert graphs.graphs and all(graphs.choosing_graphs[choosing][0] for choosing in (1, 2))
        assert llm.stepper.cache.used_pages() == 0
