"""The table of token rules on the host: masks, refusals, what a slot's row holds (no GPU needed)."""

import math

import numpy as np
import pytest
import torch

from tesseract_b200.sampling.rules import BIASES, MASK, MAX_BIASES, PENALTIES, TokenRules, mask_words, pack_mask


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 100])
def test_masks_are_bits_in_order(vocab):
    allowed = sorted({0, vocab // 2, vocab - 1})
    words = pack_mask(allowed, vocab)
    assert words.dtype == np.int32 and words.shape == (mask_words(vocab),)
    assert [t for t in range(mask_words(vocab) * 32) if int(words[t // 32]) >> t % 32 & 1] == allowed
    assert not pack_mask([], vocab).any()
    truth = np.zeros(vocab, dtype=bool)
    truth[allowed] = True
    assert np.array_equal(pack_mask(truth, vocab), words)


def test_masks_refuse_what_is_no_token():
    for allowed in ([-1], [100], [0.5], np.array([3, 100]), np.zeros(99, dtype=bool)):
        with pytest.raises(ValueError):
            pack_mask(allowed, 100)


def test_a_slots_row():
    rules = TokenRules(3, 100, "cpu", biases=4)
    assert not rules.table[:, 0].any()
    rules.set(1, repetition=1.5, presence=-0.25, frequency=2.0, biases={7: 1.0, 99: -math.inf}, allowed=[1, 99])
    row = rules.table[1]
    assert row[0].item() == PENALTIES | BIASES | MASK and row[1].item() == 2
    assert row[2:5].view(torch.float32).tolist() == [1.5, -0.25, 2.0]
    assert rules.bias_ids[1, :2].tolist() == [7, 99] and rules.biases[1, :2].tolist() == [1.0, -math.inf]
    rules.set(1)                                             # (in place of what it had)
    assert rules.table[1, :2].tolist() == [0, 0]
    assert not rules.table[0, 0] and not rules.table[2, 0]
    rules.set_mask(2, pack_mask([5], 100))
    assert rules.table[2, 0].item() == MASK


def test_refusals():
    for arguments in ((0, 10), (1, 0), (1, 10, "cpu", -1), (1, 10, "cpu", MAX_BIASES + 1)):
        with pytest.raises(ValueError):
            TokenRules(*arguments[:2], *(arguments[2:] or ("cpu",)))
    rules = TokenRules(2, 10, "cpu", biases=2)
    for slot, given in ((2, {}), (-1, {}), (0, {"repetition": 0.0}), (0, {"repetition": -1.0}), (0, {"presence": math.inf}),
                        (0, {"frequency": math.nan}), (0, {"biases": {10: 1.0}}), (0, {"biases": {-1: 1.0}}),
                        (0, {"biases": {0: math.nan}}), (0, {"biases": {0: math.inf}}), (0, {"biases": {0: 1.0, 1: 1.0, 2: 1.0}}),
                        (0, {"allowed": [10]}), (0, {"biases": {0: 1e39}}), (0, {"presence": 1e39}), (0, {"repetition": 1e-60})):
        with pytest.raises(ValueError):
            rules.set(slot, **given)
        assert not rules.table.any()                         # (a refused call leaves the rules as they were)
    with pytest.raises(ValueError):
        rules.set_biases(torch.tensor([[1, 1], [0, 1]]), torch.zeros(2, 2))
    with pytest.raises(ValueError):
        rules.set_biases(torch.tensor([[1, 2, 3], [0, 1, 2]]), torch.zeros(2, 3))
    with pytest.raises(ValueError):
        rules.set_masks(torch.zeros(2, 3, dtype=torch.int32))
    with pytest.raises(ValueError):
        rules.set_mask(0, np.zeros(2, dtype=np.int32))


def test_a_slots_history_may_be_cleared():
    rules = TokenRules(3, 100, "cpu")
    rules.seen.fill_(-1)
    rules.counts.fill_(4)
    rules.clear(1)
    assert not rules.seen[1].any() and not rules.counts[1].any()
    assert (rules.counts[[0, 2]] == 4).all() and (rules.seen[[0, 2]] == -1).all()
    with pytest.raises(ValueError):
        rules.clear(3)
