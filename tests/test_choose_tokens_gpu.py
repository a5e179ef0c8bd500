"""The choice of a token a row against the definition in 64 bits.

Tolerances: none, tokens are equal.  Scaled logits and distances are single operations in 32 bits, so both sides have the same; weights
and their sums are in 64 bits on both sides, within 2^-40 of each other, and the draws are random: that one falls between the two
sides' borders happens once in 10^6 rows of 10^5 tokens."""

import math

import numpy as np
import pytest
import torch

from tesseract_b200 import kernels
from tesseract_b200.sampling.rules import TokenRules
from tests import token_choice_plain as plain
from tests.test_token_rules_gpu import cuda, made_rules, shaped_rows

pytestmark = pytest.mark.gpu


def run(x, temperature, draw, top_k=None, top_p=None, min_p=None, rules=None, slots=None):
    rows = x.shape[0]
    whole = lambda v, dtype: cuda(np.broadcast_to(v, (rows,)).copy(), dtype) if v is not None else None  # noqa: E731
    out = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    got = kernels.choose_tokens(x, whole(temperature, torch.float32), whole(draw, torch.float64), out, top_k=whole(top_k, torch.int32),
                                top_p=whole(top_p, torch.float64), min_p=whole(min_p, torch.float64), rules=rules, slots=slots)
    assert got is out
    return got.cpu().tolist()


def check(x, temperature, draw, top_k=None, top_p=None, min_p=None, logits=None):
    """``x`` on the host; ``logits``: the same on the device in another layout."""
    rows = x.shape[0]
    logits = torch.from_numpy(x).cuda() if logits is None else logits
    got = run(logits, temperature, draw, top_k, top_p, min_p)
    one = lambda v, r, default: default if v is None else np.broadcast_to(v, (rows,))[r]  # noqa: E731
    want = [plain.choose(x[r], one(temperature, r, 0), one(draw, r, 0), int(one(top_k, r, 0)), float(one(top_p, r, 1.0)),
                         float(one(min_p, r, 0.0))) for r in range(rows)]
    assert got == want


SETTINGS = [dict(), dict(top_k=1), dict(top_k=5), dict(top_k=50, top_p=0.9), dict(top_p=0.5), dict(top_p=0.9), dict(top_p=0.999999),
            dict(top_p=1e-9), dict(min_p=0.05), dict(min_p=1.0), dict(min_p=1e-30), dict(top_k=1000, top_p=0.95, min_p=0.001),
            dict(top_k=20000), dict(top_k=20000, top_p=0.8)]


@pytest.mark.parametrize("vocab", [1, 2, 3, 5, 31, 32, 33, 257, 1000, 2049, 8192, 16385, 50257, 128256, 151936, 262144])
@pytest.mark.parametrize("settings", SETTINGS, ids=str)
def test_sizes_and_cuts(vocab, settings):
    rng = np.random.RandomState(vocab + len(str(settings)))
    rows = 5
    x = (rng.randn(rows, vocab) * np.array([0.5, 1.5, 2.5, 4.0, 9.0])[:, None]).astype(np.float32)
    check(x, np.array([0.0, 1.7, 1.0, 0.7, 0.3]), rng.rand(rows), **settings)
    check(x, 1.0, rng.rand(rows), **settings)


@pytest.mark.parametrize("rows", [1, 2, 7, 18, 19, 37, 64, 149, 300])
def test_rows_of_every_kind_beside_each_other(rows):
    rng = np.random.RandomState(rows)
    vocab = 9001
    x = (rng.randn(rows, vocab) * 2.5).astype(np.float32)
    check(x, rng.choice([0.0, 0.5, 1.0, 2.0], rows), rng.rand(rows), rng.choice([0, 1, 3, 40, 3000, 9001, 20000], rows),
          rng.choice([1.0, 0.9, 0.3], rows), rng.choice([0.0, 0.01, 0.2], rows))


@pytest.mark.parametrize("settings", SETTINGS, ids=str)
@pytest.mark.parametrize("step", [0.5, 4.0, 100.0])
@pytest.mark.parametrize("vocab", [33, 5000, 128256])
def test_equal_logits(vocab, settings, step):
    """Few distinct logits: equal ones rank by their ids, within a cut too."""
    rng = np.random.RandomState(int(step * 2) + vocab)
    x = (np.round(rng.randn(4, vocab) * 2.5 / step) * step).astype(np.float32)
    check(x, 1.0, rng.rand(4), **settings)
    check(x, 3.0, rng.rand(4), **settings)


@pytest.mark.parametrize("vocab", [1, 64, 20000, 128256])
def test_all_logits_equal_and_draws_at_the_ends(vocab):
    x = np.zeros((4, vocab), dtype=np.float32) - 3.5
    draws = np.array([0.0, 0.5, 0.25, 1.0 - 2.0 ** -53])
    for settings in SETTINGS:
        check(x, 1.0, draws, **settings)
    x[:, vocab // 2] = 4.0
    for settings in SETTINGS:
        check(x, 1.0, np.array([0.0, 1e-12, 0.999, 1.0 - 2.0 ** -53]), **settings)


@pytest.mark.parametrize("rows", [3, 32])
@pytest.mark.parametrize("spread", [0.05, 0.8, 1.2, 30.0])
def test_much_of_the_vocabulary_kept(rows, spread):
    """More is kept than one block lists, call behind call."""
    rng = np.random.RandomState(rows)
    x = (rng.randn(rows, 128256) * spread).astype(np.float32)
    x[1] += (np.arange(128256) == 777) * 20.0                # one far above the others
    x[2, :64128] = -1e30                                     # half far below
    for settings in (dict(top_p=0.95), dict(top_p=0.3), dict(top_k=30000), dict(min_p=0.05), dict(top_k=60000, top_p=0.7, min_p=0.01)):
        for temperature in (1.5, 20.0):
            check(x, temperature, rng.rand(rows), **settings)


@pytest.mark.parametrize("allowed", [1, 2, 40, 0.01, 0.5])
@pytest.mark.parametrize("vocab", [100, 50257, 128256])
def test_masked_rows(vocab, allowed):
    rng = np.random.RandomState(vocab)
    x = (rng.randn(6, vocab) * 3).astype(np.float32)
    for row in range(6):
        left = rng.permutation(vocab)[:allowed if isinstance(allowed, int) else max(1, int(allowed * vocab))]
        gone = np.ones(vocab, dtype=bool)
        gone[left] = False
        x[row, gone] = -np.inf
    for settings in SETTINGS:
        check(x, np.array([0.0, 0.5, 1.0, 1.0, 1.0, 1.5]), rng.rand(6), **settings)


def test_rows_without_a_token():
    x = np.zeros((8, 3000), dtype=np.float32)
    x[1] = -np.inf
    x[2, 77] = np.nan
    x[3, 2999] = np.inf
    x[4] = np.nan
    x[5, 1:] = -np.inf                                       # one is left
    x[6] = -3.4e38                                           # the type's lowest values are logits as others
    x[7, 5] = 3.4e38
    for temperature in (0.0, 1.0):
        for settings in SETTINGS:
            check(x, temperature, np.linspace(0, 0.99, 8), **settings)
            got = run(torch.from_numpy(x).cuda(), temperature, np.linspace(0, 0.99, 8), **settings)
            assert got[1:5] == [-1] * 4 and got[5] == 0 and got[7] == 5 and min(got[0], got[6]) >= 0


@pytest.mark.parametrize("vocab", [3, 100, 20000, 128256])
def test_a_draw_of_nothing_takes_the_first_token_that_weighs_anything(vocab):
    x = np.zeros((4, vocab), dtype=np.float32)
    for row, low in enumerate((-np.inf, -3.4028235e38, -1e4, -1500.0)):
        x[row, :vocab - 2] = low
    for settings in (dict(), dict(top_k=vocab - 1), dict(top_p=0.9)):
        check(x, 1.0, 0.0, **settings)
        assert run(torch.from_numpy(x).cuda(), 1.0, 0.0, **settings) == [vocab - 2] * 4


@pytest.mark.parametrize("temperature", [1e-40, 1e-38, 1e-30, 1e-6, 1e-3, 30.0, 1e6, 1e30, 3e38])
def test_temperatures_far_from_one(temperature):
    rng = np.random.RandomState(7)
    x = (rng.randn(5, 4000) * 3).astype(np.float32)
    x[0, :50] = -np.inf
    x[1] -= 50
    x[2] = np.round(x[2])
    for settings in (dict(), dict(top_p=0.9), dict(top_k=30), dict(min_p=0.3)):
        check(x, temperature, rng.rand(5), **settings)


@pytest.mark.parametrize("apart", [1, 2, 3, 4, 7, 64])
def test_rows_apart_and_off_their_alignment(apart):
    rng = np.random.RandomState(apart)
    vocab = 7001
    x = (rng.randn(6, vocab) * 2.5).astype(np.float32)
    store = torch.full((6, vocab + 2 * apart), 50.0, device="cuda")
    store[:, :apart] = float("nan")                          # (what lies beside the rows is nothing of theirs)
    logits = store[:, apart:apart + vocab]
    logits.copy_(torch.from_numpy(x))
    for settings in (dict(), dict(top_p=0.9), dict(top_k=30)):
        check(x, np.array([0.0, 1, 1, 1, 1, 2.0]), rng.rand(6), **settings, logits=logits)


@pytest.mark.parametrize("vocab", [33, 1000, 50257, 128256])
@pytest.mark.parametrize("rows, biases", [(1, 0), (9, 5), (30, 200)])
def test_under_rules(vocab, rows, biases):
    """The same token as of the logits that ``shape_logits`` writes, and as of the definition."""
    rng = np.random.RandomState(vocab + rows)
    slots = min(rows + 2, 9)
    rules, wanted, seen, counts = made_rules(rng, slots, vocab, biases)
    x = (rng.randn(rows, vocab) * 3).astype(np.float32)
    at = rng.randint(-1, slots + 1, rows)
    shaped = shaped_rows(x, at, wanted, seen, counts)[0].astype(np.float32)
    for r in range(rows):                                    # (NaN where the mask does not allow the token is nothing)
        if 0 <= at[r] < slots and wanted[at[r]][2] is not None and not wanted[at[r]][2].all():
            x[r, np.flatnonzero(~wanted[at[r]][2])[0]] = np.nan
    logits = torch.from_numpy(x).cuda()
    temperature, draws = rng.choice([0.0, 0.7, 1.0], rows), rng.rand(rows)
    for settings in (dict(), dict(top_k=20), dict(top_p=0.9), dict(min_p=0.05), dict(top_k=2000, top_p=0.99)):
        got = run(logits, temperature, draws, **settings, rules=rules, slots=cuda(at))
        assert got == run(kernels.shape_logits(logits, torch.empty_like(logits), rules, cuda(at)), temperature, draws, **settings)
        assert got == [plain.choose(shaped[r], temperature[r], draws[r], **settings) for r in range(rows)]


def test_a_row_has_the_token_that_it_has_alone():
    rng = np.random.RandomState(11)
    rows, vocab = 200, 30000
    logits = torch.from_numpy((rng.randn(rows, vocab) * 2).astype(np.float32)).cuda()
    draws = rng.rand(rows)
    for settings in (dict(), dict(top_p=0.95), dict(top_k=100), dict(min_p=0.02)):
        together = run(logits, 1.0, draws, **settings)
        for r in range(0, rows, 17):
            assert run(logits[r:r + 1], 1.0, draws[r:r + 1], **settings) == [together[r]]
        for _ in range(3):
            assert run(logits, 1.0, draws, **settings) == together


def test_the_tokens_of_the_samplers_that_were_there():
    """A row without a cut as ``kernels.sample``, one with top-p as the host's sampler."""
    from tesseract_b200.sampling import sample_top_p_host

    rng = np.random.RandomState(12)
    for rows, vocab in ((3, 100), (12, 32000), (40, 128256)):
        x = (rng.randn(rows, vocab) * 2.5).astype(np.float32)
        logits, temperature, draws = torch.from_numpy(x).cuda(), rng.choice([0.0, 0.6, 1.0, 1.4], rows), rng.rand(rows)
        want = kernels.sample(logits, cuda(temperature, torch.float32), cuda(draws, torch.float64),
                              torch.empty(rows, dtype=torch.int32, device="cuda")).cpu().tolist()
        assert run(logits, temperature, draws) == want
        assert run(logits, temperature, draws, top_p=0.9) == [sample_top_p_host(x[r], temperature[r], 0.9, draws[r]) for r in range(rows)]


def test_captured_and_on_two_streams():
    """A captured call replays on what its inputs hold by then, and calls on two streams do not disturb each other."""
    rng = np.random.RandomState(13)
    rows, vocab = 8, 20000
    logits = torch.zeros(rows, vocab, device="cuda")
    temperature, draws = torch.ones(rows, device="cuda"), torch.zeros(rows, dtype=torch.float64, device="cuda")
    top_p = torch.full((rows,), 0.9, dtype=torch.float64, device="cuda")
    outs = [torch.empty(rows, dtype=torch.int32, device="cuda") for _ in range(2)]
    kernels.choose_tokens(logits, temperature, draws, outs[0], top_p=top_p)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph, out in zip(graphs, outs):
        with torch.cuda.graph(graph):
            kernels.choose_tokens(logits, temperature, draws, out, top_p=top_p)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        x, u = (rng.randn(rows, vocab) * 2.5).astype(np.float32), rng.rand(rows)
        logits.copy_(torch.from_numpy(x))
        draws.copy_(torch.from_numpy(u))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        want = [plain.choose(x[r], 1.0, u[r], top_p=0.9) for r in range(rows)]
        assert outs[0].cpu().tolist() == want and outs[1].cpu().tolist() == want


def test_refusals():
    x, t, u = torch.zeros(2, 10, device="cuda"), torch.ones(2, device="cuda"), torch.zeros(2, dtype=torch.float64, device="cuda")
    out = torch.empty(2, dtype=torch.int32, device="cuda")
    rules = TokenRules(2, 10, "cuda")
    for arguments, keywords in (
            ((x.half(), t, u, out), {}), ((x, t.double(), u, out), {}), ((x, t, u.float(), out), {}), ((x, t, u, out.long()), {}),
            ((x, t[:1], u, out), {}), ((x[0], t, u, out), {}), ((x.t().contiguous().t(), t, u, out), {}), ((x[:, :0], t, u, out), {}),
            ((x, t, u, out), {"top_k": u}), ((x, t, u, out), {"top_p": t}), ((x, t, u, out), {"min_p": t}),
            ((x, t, u, out), {"top_p": u[:1]}), ((x, t, u, out), {"slots": out}), ((x, t, u, out), {"rules": rules}),
            ((x, t, u, out), {"rules": TokenRules(2, 11, "cuda"), "slots": out}), ((x, t, u, out.cpu()), {}),
            ((x, None, u, out), {}), ((torch.zeros(2, 262145, device="cuda"), t, u, out), {}),
            ((x, t, u, out), {"rules": TokenRules(2, 10, "cpu"), "slots": out}), ((x.cpu(), t, u, out), {}),
            ((torch.zeros(2, 19, device="cuda").as_strided((2, 10), (9, 1)), t, u, out), {})):
        with pytest.raises(kernels.KernelError):
            kernels.choose_tokens(*arguments, **keywords)
    none = torch.empty(0, 10, device="cuda")
    assert kernels.choose_tokens(none, t[:0], u[:0], out[:0]).numel() == 0
