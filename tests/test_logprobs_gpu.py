"""Log probabilities, entropy and alternatives against the definition in 64 bits.

Tolerances.  With u = 2^-24: a log probability is (x_t - m) - ln S, two roundings of numbers up to its own size and of ln S, plus the
relative error of S, which is a sum of V positive terms in at most 16 * (V / 8192) + 25 additions a term, each term within 4 u
of relative error beyond the argument's rounding, u |d| log2(e) with |d| up to 60 weighed by e^d (|d| e^d <= 0.37): below
(16 V / 8192 + 35) u.  The entropy adds T / S, whose terms are |d| e^d <= 0.37 each: errors of T of (16 V / 8192 + 35) u T.
Both are checked at (16 V / 8192 + 60) u * (1 + |value|) with |value| the largest magnitude that enters the difference.
"""

import math

import pytest
import torch

from tesseract_b200 import kernels

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def definition(logits, tokens, k):
    x = logits.double().cpu()
    logs = x - torch.logsumexp(x, dim=1, keepdim=True)
    p = torch.exp(logs)
    entropy = -torch.where(p > 0, p * logs, torch.zeros((), dtype=torch.float64)).sum(dim=1)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
    return logs.gather(1, tokens.long().cpu()[:, None])[:, 0], entropy, logs.gather(1, order), order


def check(logits, tokens, k):
    got = kernels.token_logprobs(logits, tokens, k)
    want = definition(logits, tokens, k)
    vocab = logits.shape[1]
    finite = logits.double()[torch.isfinite(logits)]
    span = float(finite.abs().max()) if finite.numel() else 0.0
    bound = (16 * vocab / 8192 + 60) * U * (1 + 2 * span + math.log(vocab))
    for name, g, w in zip(("logprob", "entropy", "values"), got, want):
        g = g.double().cpu()
        assert torch.equal(torch.isinf(g), torch.isinf(w)), name
        there = torch.isfinite(w)
        assert float((g - w)[there].abs().max() if bool(there.any()) else 0.0) <= bound, name
    assert got[3].dtype == torch.int32
    assert torch.equal(got[3].cpu().long(), want[3])
    return got


def tokens_for(rows, vocab, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(0, vocab, (rows,), generator=gen, dtype=torch.int32).cuda()


@pytest.mark.parametrize("vocab", [1, 2, 3, 5, 31, 64, 257, 8191, 8192, 8193, 16384, 16390, 50257, 128256])
@pytest.mark.parametrize("rows, k", [(1, 1), (3, 20), (5, 64), (40, 7), (2, 0)])
def test_sizes(rows, vocab, k):
    gen = torch.Generator(device="cuda").manual_seed(vocab + rows)
    logits = torch.randn(rows, vocab, generator=gen, device="cuda") * 3
    check(logits, tokens_for(rows, vocab), min(k, vocab))


@pytest.mark.parametrize("apart", [1, 2, 3, 4, 7])
@pytest.mark.parametrize("vocab", [257, 8190, 33001])
def test_rows_apart_and_off_the_boundary(vocab, apart):
    gen = torch.Generator(device="cuda").manual_seed(apart)
    whole = torch.full((6, vocab + apart), math.inf, device="cuda")       # what lies between rows is not read into a sum
    whole[:, :vocab] = torch.randn(6, vocab, generator=gen, device="cuda")
    check(whole[:, :vocab], tokens_for(6, vocab), 9)
    whole[:, 0] = math.nan
    whole[:, 1:] = torch.randn(6, vocab + apart - 1, generator=gen, device="cuda")
    check(whole[:, 1:], tokens_for(6, vocab), 9)


@pytest.mark.parametrize("rows, vocab", [(1, 3000001), (300, 1100003)])
def test_vocabularies_of_more_groups_than_are_kept(rows, vocab):
    gen = torch.Generator(device="cuda").manual_seed(rows)
    logits = torch.randn(rows, vocab, generator=gen, device="cuda")
    tokens = tokens_for(rows, vocab)
    got = kernels.token_logprobs(logits, tokens, 40)
    for r in {0, rows // 2, rows - 1}:
        logs = torch.log_softmax(logits[r].double(), dim=0)
        order = torch.sort(logits[r], descending=True, stable=True).indices[:40]
        bound = (16 * vocab / 4096 + 60) * U * 30
        assert torch.equal(got[3][r].long(), order)
        assert float((got[2][r].double() - logs[order]).abs().max()) <= bound
        assert abs(float(got[0][r]) - float(logs[int(tokens[r])])) <= bound
        assert abs(float(got[1][r]) + float((logs.exp() * logs).sum())) <= bound


@pytest.mark.parametrize("rows", [140, 150, 290, 300, 600])
def test_every_size_of_block(rows):
    gen = torch.Generator(device="cuda").manual_seed(rows)
    logits = torch.randn(rows, 9001, generator=gen, device="cuda") * 2
    check(logits, tokens_for(rows, 9001), 17)


@pytest.mark.parametrize("rows", [1, 30, 400])
def test_the_same_numbers_at_every_split(rows):
    """How many blocks share a row depends on the rows: alternatives are the same tokens whichever."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    one = torch.randn(1, 40000, generator=gen, device="cuda") * 2
    got = check(one.expand(rows, -1).contiguous(), torch.full((rows,), 77, dtype=torch.int32, device="cuda"), 32)
    for part in got:
        assert bool((part == part[:1]).all())


@pytest.mark.parametrize("k", [1, 20, 64])
@pytest.mark.parametrize("vocab", [300, 8192, 30000])
def test_ties_go_to_the_lowest_id(vocab, k):
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    few = torch.randint(-3, 4, (4, vocab), generator=gen, device="cuda").float()
    check(few, tokens_for(4, vocab), k)
    check(torch.zeros(3, vocab, device="cuda"), tokens_for(3, vocab), k)
    zeros = torch.zeros(2, vocab, device="cuda")
    zeros[:, ::2] = -0.0
    check(zeros, tokens_for(2, vocab), k)
    steps = (torch.arange(vocab, device="cuda") // 700).float().expand(2, -1).contiguous()
    check(steps, tokens_for(2, vocab), k)


@pytest.mark.parametrize("k", [1, 33, 64])
def test_orders_that_defeat_the_bound(k):
    """Logits that rise with the id (every chunk's are all above what came before), that fall, and one high block."""
    vocab = 70001
    up = torch.linspace(-20, 20, vocab, device="cuda").expand(2, -1).contiguous()
    check(up, tokens_for(2, vocab), k)
    check(up.flip(1).contiguous(), tokens_for(2, vocab), k)
    block = torch.full((300, vocab), -5.0, device="cuda")
    block[:, 40000:40300] = 5.0 + torch.arange(300, device="cuda") / 64
    check(block, tokens_for(300, vocab), k)


@pytest.mark.parametrize("allowed", [1, 2, 10, 63, 64, 65, 500])
def test_masked_vocabulary(allowed):
    vocab = 20011
    gen = torch.Generator(device="cuda").manual_seed(allowed)
    logits = torch.full((5, vocab), -math.inf, device="cuda")
    for r in range(5):
        where = torch.randperm(vocab, generator=gen, device="cuda")[:allowed]
        logits[r, where] = torch.randn(allowed, generator=gen, device="cuda") * 4
    tokens = tokens_for(5, vocab)
    tokens[0] = int(logits[0].argmax())
    got = check(logits, tokens, 64)
    assert math.isfinite(float(got[0][0]))


def test_the_types_lowest_value_as_a_mask():
    logits = torch.full((3, 9000), torch.finfo(torch.float32).min, device="cuda")
    logits[0, 17] = 2.0
    logits[1, [5, 8000]] = torch.tensor([1.0, 3.0], device="cuda")
    got = kernels.token_logprobs(logits, torch.tensor([17, 5, 0], dtype=torch.int32, device="cuda"), 3)
    assert float(got[0][0]) == 0.0 and float(got[1][0]) == 0.0
    assert got[3].tolist() == [[17, 0, 1], [8000, 5, 0], [0, 1, 2]]
    assert abs(float(got[0][2]) + math.log(9000)) < 1e-5
    assert abs(float(got[1][2]) - math.log(9000)) < 1e-5


def test_a_certain_row_and_a_large_shift():
    logits = torch.randn(2, 5000, device="cuda")
    logits[0, 3] = 200.0
    logits[1] += 1.0e4
    check(logits, torch.tensor([3, 9], dtype=torch.int32, device="cuda"), 4)


@pytest.mark.parametrize("poison", [math.nan, math.inf])
def test_nan_and_infinity_stay_in_their_row(poison):
    logits = torch.randn(4, 12345, device="cuda")
    logits[2, 11111] = poison
    tokens = tokens_for(4, 12345)
    got = kernels.token_logprobs(logits, tokens, 8)
    assert math.isnan(float(got[0][2])) and math.isnan(float(got[1][2])) and bool(torch.isnan(got[2][2]).all())
    assert bool(((got[3] >= 0) & (got[3] < 12345)).all())
    keep = [0, 1, 3]
    want = definition(logits[keep], tokens[keep], 8)
    assert torch.equal(got[3][keep].cpu().long(), want[3])
    assert bool(torch.isfinite(got[0][keep]).all())


def test_a_row_with_nothing_allowed():
    logits = torch.full((2, 3000), -math.inf, device="cuda")
    logits[1, 5] = 0.0
    got = kernels.token_logprobs(logits, torch.tensor([1, 5], dtype=torch.int32, device="cuda"), 5)
    assert math.isnan(float(got[0][0])) and math.isnan(float(got[1][0]))
    assert got[3].tolist() == [[0, 1, 2, 3, 4], [5, 0, 1, 2, 3]]
    assert float(got[0][1]) == 0.0


def test_tokens_outside_the_vocabulary():
    logits = torch.randn(3, 100, device="cuda")
    got = kernels.token_logprobs(logits, torch.tensor([-1, 100, 99], dtype=torch.int32, device="cuda"), 2)
    assert torch.isnan(got[0]).tolist() == [True, True, False]
    assert bool(torch.isfinite(got[1]).all())


def test_no_rows():
    got = kernels.token_logprobs(torch.empty(0, 50, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), 4)
    assert [tuple(t.shape) for t in got] == [(0,), (0,), (0, 4), (0, 4)]


def test_refusals():
    logits, tokens = torch.randn(4, 50, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad in [(logits.bfloat16(), tokens, 1), (logits, tokens.long(), 1), (logits, tokens[:3], 1), (logits, tokens, 51),
                (logits, tokens, 65), (logits, tokens, -1), (logits[:, ::2], tokens, 1), (logits.cpu(), tokens, 1),
                (logits, tokens.cpu(), 1), (logits[0], tokens, 1)]:
        with pytest.raises(kernels.KernelError):
            kernels.token_logprobs(*bad)


@pytest.mark.parametrize("rows", [150, 300])
@pytest.mark.parametrize("vocab", [262143, 262144, 262145, 262161])
def test_either_side_of_the_groups_that_a_block_keeps(rows, vocab):
    """One block a row, of 512 and of 256 threads: up to 262,144 logits of a part each group is one chunk's."""
    gen = torch.Generator(device="cuda").manual_seed(rows + vocab)
    logits = torch.randn(rows, vocab + 3, generator=gen, device="cuda")[:, :vocab]
    logits[:, -1] = 9.0                                # (the last logit is the largest)
    tokens = tokens_for(rows, vocab)
    got = kernels.token_logprobs(logits, tokens, 40)
    for r in (0, 1, 2, 3, rows - 1):
        logs = torch.log_softmax(logits[r].double(), dim=0)
        order = torch.sort(logits[r], descending=True, stable=True).indices[:40]
        bound = (16 * vocab / 4096 + 60) * U * 30
        assert torch.equal(got[3][r].long(), order) and int(order[0]) == vocab - 1
        assert float((got[2][r].double() - logs[order]).abs().max()) <= bound
        assert abs(float(got[0][r]) - float(logs[int(tokens[r])])) <= bound
        assert abs(float(got[1][r]) + float((logs.exp() * logs).sum())) <= bound


@pytest.mark.parametrize("rows", [3, 200])
def test_on_another_stream_and_behind_its_inputs(rows):
    logits = torch.randn(rows, 30011, device="cuda") * 2
    tokens = tokens_for(rows, 30011)
    want = kernels.token_logprobs(logits, tokens, 12)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late, late_tokens = torch.zeros_like(logits), torch.zeros_like(tokens)
        torch.cuda._sleep(2_000_000)
        late.copy_(logits)
        late_tokens.copy_(tokens)
        got = kernels.token_logprobs(late, late_tokens, 12)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
