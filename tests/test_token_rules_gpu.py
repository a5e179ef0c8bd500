"""Histories of tokens and logits under rules, against numpy in 64 bits.

Tolerances.  Histories are whole numbers: equal.  A shaped logit is computed in 64 bits (at most five operations, each within 2^-53 of
its result, whose size is at most the sum of what goes in: below 2^-50 of that sum) and rounded once to 32 bits: within 2^-24 of its
value, and 2^-50 of the sum of the magnitudes that went in."""

import numpy as np
import pytest
import torch

from tesseract_b200 import kernels
from tesseract_b200.sampling.rules import TokenRules, pack_mask
from tests import token_choice_plain as plain

pytestmark = pytest.mark.gpu


def cuda(values, dtype=torch.int32):
    return torch.tensor(np.asarray(values), dtype=dtype).cuda()


def bits(words, vocab):
    return np.unpackbits(np.ascontiguousarray(words.cpu().numpy()).view(np.uint8), axis=1, bitorder="little")[:, :vocab] != 0


def check_history(rules, seen, counts):
    assert np.array_equal(rules.counts.cpu().numpy(), counts)
    assert np.array_equal(bits(rules.seen, rules.vocab), seen)
    # (nothing behind the vocabulary)
    assert int(rules._counts[:, rules.vocab:].abs().sum()) == 0
    assert not np.unpackbits(rules._seen.cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, rules.vocab:].any()


@pytest.mark.parametrize("vocab", [1, 2, 31, 32, 33, 127, 1000, 8193, 50257, 128256])
@pytest.mark.parametrize("lengths", [[0], [1], [5, 0, 1], [3000, 17, 0, 40, 1, 1, 2, 9000]])
def test_prompts_and_answers(vocab, lengths):
    rng = np.random.RandomState(vocab + len(lengths))
    slots = len(lengths) + 2
    rules = TokenRules(slots, vocab, "cuda")
    seen, counts = np.zeros((slots, vocab), dtype=bool), np.zeros((slots, vocab), dtype=np.int32)
    for restart in (True, False, True):
        at = rng.permutation(slots)[:len(lengths)]
        parts = [(rng.rand(n) ** 3 * vocab).astype(np.int32) for n in lengths]
        prompts = [int(rng.randint(0, n + 2)) for n in lengths]
        kernels.note_tokens(rules, cuda(at), cuda(np.concatenate(parts)), starts=cuda(np.concatenate([[0], np.cumsum(lengths)])),
                            prompts=cuda(prompts), restart=restart)
        for slot, part, prompt in zip(at, parts, prompts):
            plain.note(seen, counts, slot, part, prompt, restart)
        check_history(rules, seen, counts)


@pytest.mark.parametrize("rows", [1, 2, 33, 300])
def test_a_token_a_row(rows):
    vocab, slots = 700, 7
    rng = np.random.RandomState(rows)
    rules = TokenRules(slots, vocab, "cuda")
    seen, counts = np.zeros((slots, vocab), dtype=bool), np.zeros((slots, vocab), dtype=np.int32)
    for _ in range(3):
        # (slots named by many rows, by none, and outside the table; tokens outside the vocabulary)
        at = rng.randint(-2, slots + 2, rows)
        tokens = rng.randint(-3, vocab + 3, rows)
        prompts = rng.randint(0, 2, rows)
        kernels.note_tokens(rules, cuda(at), cuda(tokens), prompts=cuda(prompts))
        for slot, token, prompt in zip(at, tokens, prompts):
            plain.note(seen, counts, slot, [token], prompt)
        check_history(rules, seen, counts)
    kernels.note_tokens(rules, cuda(at), cuda(tokens))                      # (without prompts everything is an answer's)
    for slot, token in zip(at, tokens):
        plain.note(seen, counts, slot, [token])
    check_history(rules, seen, counts)


def test_of_rows_that_begin_one_slot_anew_the_last_counts():
    rules = TokenRules(3, 100, "cuda")
    seen, counts = np.zeros((3, 100), dtype=bool), np.zeros((3, 100), dtype=np.int32)
    kernels.note_tokens(rules, cuda([1, 0, 1, 1]), cuda([5, 6, 7, 8, 9, 5]), starts=cuda([0, 2, 3, 5, 6]), restart=True)
    plain.note(seen, counts, 0, [7], 0, True)
    plain.note(seen, counts, 1, [5], 0, True)
    check_history(rules, seen, counts)


def test_starts_that_leave_the_list_name_no_tokens():
    rules = TokenRules(3, 100, "cuda")
    seen, counts = np.zeros((3, 100), dtype=bool), np.zeros((3, 100), dtype=np.int32)
    kernels.note_tokens(rules, cuda([0, 1, 2]), cuda([5, 6, 7]), starts=cuda([-4, 2, 1, 90]))
    plain.note(seen, counts, 0, [5, 6])
    plain.note(seen, counts, 2, [6, 7])
    check_history(rules, seen, counts)


def made_rules(rng, slots, vocab, biases, penalties=True, masks=True):
    """Rules of every kind: slot 0 has none, the others some."""
    rules = TokenRules(slots, vocab, "cuda", biases=biases)
    wanted = []
    for slot in range(slots):
        rule, given, allowed = None, {}, None
        if slot and penalties and slot % 3 != 0:
            rule = (float(rng.rand() + 0.6), float(rng.randn()), float(rng.randn() * 0.3))
        if slot and biases and slot % 2:
            given = {int(t): float(b) for t, b in zip(rng.permutation(vocab)[:rng.randint(0, min(biases, vocab) + 1)], rng.randn(biases) * 4)}
        if slot and masks and slot % 4 < 2:
            allowed = rng.rand(vocab) < rng.choice([0.01, 0.5, 0.99])
        keywords = dict(zip(("repetition", "presence", "frequency"), rule)) if rule else {}
        rules.set(slot, **keywords, biases=given, allowed=np.flatnonzero(allowed) if allowed is not None else None)
        wanted.append((rule, given, allowed))
    seen, counts = np.zeros((slots, vocab), dtype=bool), np.zeros((slots, vocab), dtype=np.int32)
    lengths = rng.randint(0, 2 * vocab if vocab < 500 else 1500, slots)
    parts = [(rng.rand(n) ** 2 * vocab).astype(np.int32) for n in lengths]
    prompts = [n // 2 for n in lengths]
    kernels.note_tokens(rules, cuda(range(slots)), cuda(np.concatenate(parts)), starts=cuda(np.concatenate([[0], np.cumsum(lengths)])),
                        prompts=cuda(prompts), restart=True)
    for slot in range(slots):
        plain.note(seen, counts, slot, parts[slot], prompts[slot])
    return rules, wanted, seen, counts


def shaped_rows(x, at, wanted, seen, counts):
    rows, sizes = [], []
    for row, slot in zip(x, at):
        if not 0 <= slot < len(wanted):
            rows.append(row.astype(np.float64))
            sizes.append(np.abs(rows[-1]))
            continue
        rule, given, allowed = wanted[slot]
        rows.append(plain.shaped(row, rule, seen[slot], counts[slot], given, allowed))
        size = np.abs(row.astype(np.float64)) * 2 + (abs(rule[1]) + abs(rule[2]) * counts[slot] if rule else 0.0)
        for token, bias in given.items():
            size[token] += abs(bias)
        sizes.append(size)
    return np.stack(rows), np.stack(sizes)


def check_shaped(got, want, size):
    got = got.cpu().numpy().astype(np.float64)
    there = np.isfinite(want)
    assert np.array_equal(got[~there], want[~there], equal_nan=True)
    assert (np.abs(got[there] - want[there]) <= 2.0 ** -24 * np.abs(want[there]) + 2.0 ** -50 * size[there] + 2.0 ** -149).all()


@pytest.mark.parametrize("vocab", [1, 2, 31, 32, 33, 100, 257, 4099, 50257, 128256])
@pytest.mark.parametrize("rows, biases", [(1, 0), (5, 3), (40, 300)])
@pytest.mark.parametrize("apart", [0, 1, 4])
def test_shaped_logits(vocab, rows, biases, apart):
    rng = np.random.RandomState(vocab * 3 + rows + apart)
    slots = min(rows + 2, 9)
    rules, wanted, seen, counts = made_rules(rng, slots, vocab, biases)
    x = (rng.randn(rows, vocab) * 4).astype(np.float32)
    if vocab > 3:
        x[:, 2], x[0, 3], x[-1, 1] = 0.0, -np.inf, np.nan
    at = rng.randint(-1, slots + 1, rows)
    store = torch.full((rows, vocab + apart), 7.0, device="cuda")
    logits = store[:, :vocab]
    logits.copy_(torch.from_numpy(x))
    keep = torch.full((rows, vocab + 2 * apart), 3.0, device="cuda")
    out = keep[:, apart:apart + vocab]
    want, size = shaped_rows(x, at, wanted, seen, counts)
    assert kernels.shape_logits(logits, out, rules, cuda(at)) is out
    check_shaped(out, want, size)
    assert np.array_equal(logits.cpu().numpy(), x, equal_nan=True) and bool((store[:, vocab:] == 7.0).all())
    assert bool((keep[:, :apart] == 3.0).all()) and bool((keep[:, apart + vocab:] == 3.0).all())
    kernels.shape_logits(logits, logits, rules, cuda(at))                  # in place: the same bits
    assert np.array_equal(logits.cpu().numpy(), out.cpu().numpy(), equal_nan=True) and bool((store[:, vocab:] == 7.0).all())


def test_a_bias_of_every_kind():
    vocab = 64
    rules = TokenRules(2, vocab, "cuda", biases=4)
    rules.set(1, biases={0: -float("inf"), 5: 100.0, 63: -1e-30, 7: 3.0e38}, allowed=[0, 5, 7, 9, 63])
    x = np.zeros((1, vocab), dtype=np.float32)
    x[0, 7] = 3.0e38
    got = kernels.shape_logits(cuda(x, torch.float32), torch.empty(1, vocab, device="cuda"), rules, cuda([1])).cpu().numpy()[0]
    want = np.full(vocab, -np.inf)
    want[[5, 7, 9]], want[63] = [100.0, np.inf, 0.0], np.float32(-1e-30)
    assert np.array_equal(got.astype(np.float64), want)


def test_rules_are_replaced_and_copied():
    rng = np.random.RandomState(3)
    vocab, slots = 300, 6
    rules, wanted, seen, counts = made_rules(rng, slots, vocab, 8)
    rules.copy([1, 4], [2, 0])
    for source, target in ((1, 2), (4, 0)):
        wanted[target], seen[target], counts[target] = wanted[source], seen[source], counts[source]
    rules.set(5)
    wanted[5] = (None, {}, None)
    rules.set_mask(3, pack_mask([1, 2, 299], vocab))
    only = np.zeros(vocab, dtype=bool)
    only[[1, 2, 299]] = True
    wanted[3] = (*wanted[3][:2], only)
    x = (rng.randn(slots, vocab) * 4).astype(np.float32)
    want, size = shaped_rows(x, range(slots), wanted, seen, counts)
    check_shaped(kernels.shape_logits(cuda(x, torch.float32), torch.empty(slots, vocab, device="cuda"), rules, cuda(range(slots))), want, size)
    check_history(rules, seen, counts)


def test_captured_and_on_another_stream():
    """A captured pair of calls replays on what the history, the logits and the slots hold by then."""
    rng = np.random.RandomState(5)
    vocab, slots, rows = 5000, 5, 4
    rules, wanted, seen, counts = made_rules(rng, slots, vocab, 8)
    at, tokens = cuda([-1] * rows), cuda([0] * rows)
    logits, out = torch.zeros(rows, vocab, device="cuda"), torch.empty(rows, vocab, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.note_tokens(rules, at, tokens)
        kernels.shape_logits(logits, out, rules, at)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.note_tokens(rules, at, tokens)
        kernels.shape_logits(logits, out, rules, at)
    for _ in range(3):
        x, slot, token = (rng.randn(rows, vocab) * 4).astype(np.float32), rng.randint(-1, slots, rows), rng.randint(0, vocab, rows)
        logits.copy_(torch.from_numpy(x))
        at.copy_(torch.from_numpy(slot))
        tokens.copy_(torch.from_numpy(token))
        graph.replay()
        for s, t in zip(slot, token):
            plain.note(seen, counts, s, [t])
        want, size = shaped_rows(x, slot, wanted, seen, counts)
        check_shaped(out, want, size)
        check_history(rules, seen, counts)


def test_slots_far_into_a_large_table():
    """A slot whose counts begin beyond 2^31 numbers."""
    vocab, slots = 128256, 16800
    if torch.cuda.mem_get_info()[0] < 16e9:
        pytest.skip("needs 16 GB")
    rules = TokenRules(slots, vocab, "cuda")
    assert rules.counts.stride(0) * (slots - 1) > 2 ** 31
    rules.set(slots - 1, frequency=1.0, allowed=[vocab - 1, 3])
    kernels.note_tokens(rules, cuda([slots - 1]), cuda([3, vocab - 1, 3]), starts=cuda([0, 3]), restart=True)
    got = kernels.shape_logits(torch.zeros(1, vocab, device="cuda"), torch.empty(1, vocab, device="cuda"), rules, cuda([slots - 1]))
    assert got[0, 3].item() == -2.0 and got[0, vocab - 1].item() == -1.0 and bool(torch.isinf(got[0, 4:vocab - 1]).all())


def test_refusals():
    rules = TokenRules(4, 100, "cuda", biases=2)
    x, out, at = torch.zeros(2, 100, device="cuda"), torch.empty(2, 100, device="cuda"), cuda([0, 1])
    with pytest.raises(kernels.KernelError):
        kernels.shape_logits(x, out, rules, cuda([0]))
    with pytest.raises(kernels.KernelError):
        kernels.shape_logits(x, out, rules, at.long())
    with pytest.raises(kernels.KernelError):
        kernels.shape_logits(x[:, :99], out[:, :99], rules, at)
    with pytest.raises(kernels.KernelError):
        kernels.shape_logits(x, out[:1], rules, at)
    with pytest.raises(kernels.KernelError):
        kernels.shape_logits(x.half(), out, rules, at)
    with pytest.raises(kernels.KernelError):
        kernels.shape_logits(x.t().contiguous().t(), out, rules, at)
    with pytest.raises(kernels.KernelError):
        kernels.shape_logits(x, torch.empty(2, 100), rules, at)
    with pytest.raises(kernels.KernelError):                              # rows that lie on the logits, not in their places
        both = torch.zeros(3, 100, device="cuda")
        kernels.shape_logits(both[:2], both[1:], rules, at)
    with pytest.raises(kernels.KernelError):
        kernels.note_tokens(rules, at, cuda([1]))
    with pytest.raises(kernels.KernelError):
        kernels.note_tokens(rules, at, cuda([1, 2]), starts=cuda([0, 2]))
    with pytest.raises(kernels.KernelError):
        kernels.note_tokens(rules, at, cuda([1, 2]), prompts=cuda([0]))
    with pytest.raises(kernels.KernelError):
        kernels.note_tokens(rules, at, cuda([1, 2]).float())
    # nothing to do is no error
    none = cuda(np.zeros(0))
    kernels.note_tokens(rules, none, none)
    assert kernels.shape_logits(x[:0], out[:0], rules, none).shape == (0, 100)
