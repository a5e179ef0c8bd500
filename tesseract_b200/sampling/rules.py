"""The rules that requests put on their next tokens, one slot a request, as the kernels read them.

A slot has penalties (``repetition`` divides the positive and multiplies the negative logits of tokens that the request has had,
``frequency`` is taken off for every time its answer has a token, ``presence`` off once), biases added to the logits of single tokens,
a mask of the tokens that may come next, and the history that the penalties go by (``kernels.note_tokens`` writes it).  The kernels
``shape_logits`` and ``choose_tokens`` are given a slot a row.  Not in the reference, whose requests have a temperature and top-p
(src/engine/types.rs:14-37).
"""

from __future__ import annotations

import math
from typing import Dict, Iterable, Mapping, Optional, Sequence, Union

import numpy as np
import torch

from .. import kernels
from .params import MAX_BIASES, single

PENALTIES, BIASES, MASK = 1, 2, 4


def mask_words(vocab: int) -> int:
    """int32 words of a mask: token ``t`` is bit ``t % 32`` of word ``t // 32``."""
    return -(-vocab // 32)


def pack_mask(allowed: Iterable[int], vocab: int) -> np.ndarray:
    """The mask words of the given token ids, or of truth values, one a token (an array ``[vocab]``); ids outside the vocabulary raise."""
    if isinstance(allowed, np.ndarray) and allowed.dtype == np.bool_:
        if allowed.shape != (vocab,):
            raise ValueError(f"a mask of truth values has one for each of the vocabulary's {vocab}")
        bits = np.zeros(mask_words(vocab) * 32, dtype=np.bool_)
        bits[:vocab] = allowed
        return np.packbits(bits, bitorder="little").view(np.int32)
    ids = np.asarray(allowed if isinstance(allowed, np.ndarray) else list(allowed))
    bits = np.zeros(mask_words(vocab) * 32, dtype=np.uint8)
    if ids.size:
        if ids.dtype.kind not in "iu" or int(ids.min()) < 0 or int(ids.max()) >= vocab:
            raise ValueError(f"allowed tokens are ids of the vocabulary of {vocab}")
        bits[ids] = 1
    return np.packbits(bits, bitorder="little").view(np.int32)


class TokenRules:
    """Rules and histories of ``slots`` requests over ``vocab`` tokens, with room for ``biases`` biases each.

    ``counts`` int32 ``[slots, vocab]``: how often the answer has a token; ``seen`` int32 ``[slots, words]``: a bit for every token
    of the prompt and the answer; ``masks`` likewise; ``table`` int32 ``[slots, 8]``: kinds of rules, number of biases, and the bits
    of the three penalties.  All writes are on the current stream."""

    def __init__(self, slots: int, vocab: int, device, biases: int = 0):
        if slots < 1 or vocab < 1 or not 0 <= biases <= MAX_BIASES:
            raise ValueError(f"token rules need a slot and a token at least, and have room for up to {MAX_BIASES} biases")
        self.slots, self.vocab, self.room, self.words = slots, vocab, biases, mask_words(vocab)
        self.device = torch.device(device)
        wide = -(-self.words // 4) * 4                       # (rows of words and of counts begin on 16 bytes)
        self.table = torch.zeros(slots, 8, dtype=torch.int32, device=device)
        self._seen = torch.zeros(slots, wide, dtype=torch.int32, device=device)
        self._counts = torch.zeros(slots, wide * 32, dtype=torch.int32, device=device)
        self._masks = torch.zeros(slots, wide, dtype=torch.int32, device=device)
        self.bias_ids = torch.zeros(slots, biases, dtype=torch.int32, device=device)
        self.biases = torch.zeros(slots, biases, dtype=torch.float32, device=device)
        self.seen, self.counts = self._seen[:, :self.words], self._counts[:, :vocab]
        self.masks = self._masks[:, :self.words]
        self.record = kernels.RulesRecord(None, *[t.data_ptr() for t in (self.table, self._seen, self._counts, self._masks, self.bias_ids,
                                                                        self.biases)], slots, wide, 32 * wide, biases)
        self.index = self.table.get_device()                 # (-1 on the host)
        self.history = (self._seen.data_ptr(), self._counts.data_ptr(), slots, wide, 32 * wide)
        self._host = np.zeros((slots, 8), dtype=np.int32)
        self._host[:, 2] = np.float32(1.0).view(np.int32)

    def _check(self, slot: int) -> None:
        if not 0 <= slot < self.slots:
            raise ValueError(f"slot {slot} is outside the {self.slots} of these rules")

    def _upload(self, slot: Optional[int] = None) -> None:
        if slot is None or not self.table.is_cuda:
            self.table.copy_(torch.from_numpy(self._host))
        else:
            kernels.set_rules(self.table, slot, self._host[slot].tolist())

    def set(self, slot: int, *, repetition: float = 1.0, presence: float = 0.0, frequency: float = 0.0,
            biases: Optional[Mapping[int, float]] = None, allowed: Optional[Iterable[int]] = None) -> None:
        """A slot's rules from now on, in place of those it had; its history stays (``kernels.note_tokens(..., restart=True)``)."""
        self._check(slot)
        repetition, presence, frequency = single(repetition), single(presence), single(frequency)
        if not (math.isfinite(repetition) and repetition > 0.0 and math.isfinite(presence) and math.isfinite(frequency)):
            raise ValueError("penalties must be finite, and the one for repetition positive")
        row = np.zeros(8, dtype=np.int32)
        row[2:5] = np.asarray([repetition, presence, frequency], dtype=np.float32).view(np.int32)
        if not (repetition == 1.0 and presence == 0.0 and frequency == 0.0):
            row[0] |= PENALTIES
        words = None
        if allowed is not None:
            words = pack_mask(allowed, self.vocab)
            row[0] |= MASK
        if biases:
            ids, values = np.asarray(list(biases.keys())), np.asarray([single(bias) for bias in biases.values()], dtype=np.float32)
            if ids.size > self.room:
                raise ValueError(f"{ids.size} biases, and room for {self.room}")
            self._check_biases(ids[None], values[None])
            row[0] |= BIASES
            row[1] = ids.size
            self.bias_ids[slot, :ids.size] = torch.from_numpy(ids.astype(np.int32)).to(self.device)
            self.biases[slot, :ids.size] = torch.from_numpy(values).to(self.device)
        if words is not None:
            self.masks[slot] = torch.from_numpy(words).to(self.device)
        if not np.array_equal(row, self._host[slot]):
            self._host[slot] = row
            self._upload(slot)

    def _check_biases(self, ids: np.ndarray, values: np.ndarray) -> None:
        if ids.size == 0:
            return
        if ids.dtype.kind not in "iu" or int(ids.min()) < 0 or int(ids.max()) >= self.vocab:
            raise ValueError(f"biases name tokens of the vocabulary of {self.vocab}")
        if np.isnan(values).any() or np.isposinf(values).any():
            raise ValueError("biases must be finite (or -inf, which rules a token out)")
        ranked = np.sort(ids, axis=1)
        if (ranked[:, 1:] == ranked[:, :-1]).any():
            raise ValueError("a slot's biases name a token once")

    def set_biases(self, ids: torch.Tensor, values: torch.Tensor) -> None:
        """Biases of all slots: ``ids`` and ``values`` ``[slots, n]``, no token twice in a slot."""
        if ids.shape != values.shape or ids.dim() != 2 or ids.shape[0] != self.slots or ids.shape[1] > self.room:
            raise ValueError(f"biases are [{self.slots}, up to {self.room}] ids and values")
        n = ids.shape[1]
        self._check_biases(ids.cpu().numpy(), values.float().cpu().numpy())
        self.bias_ids[:, :n] = ids
        self.biases[:, :n] = values
        self._host[:, 0] = self._host[:, 0] | BIASES if n else self._host[:, 0] & ~BIASES
        self._host[:, 1] = n
        self._upload()

    def set_masks(self, words: torch.Tensor) -> None:
        """The masks of all slots, int32 words ``[slots, words]`` (:func:`pack_mask`)."""
        if words.shape != self.masks.shape or words.dtype != torch.int32:
            raise ValueError(f"masks are int32 [{self.slots}, {self.words}]")
        self.masks.copy_(words)
        self._host[:, 0] |= MASK
        self._upload()

    def set_mask(self, slot: int, words: Union[np.ndarray, torch.Tensor]) -> None:
        """One slot's mask (:func:`pack_mask`)."""
        self._check(slot)
        words = torch.as_tensor(words)
        if words.shape != (self.words,) or words.dtype != torch.int32:
            raise ValueError(f"a mask is {self.words} int32 words")
        self.masks[slot].copy_(words, non_blocking=True)
        if not self._host[slot, 0] & MASK:
            self._host[slot, 0] |= MASK
            self._upload(slot)

    def clear(self, slot: int) -> None:
        """A slot's history begins anew."""
        self._check(slot)
        self._seen[slot].zero_()
        self._counts[slot].zero_()

    def copy(self, sources: Sequence[int], targets: Sequence[int]) -> None:
        """Rules and histories of slots into others, in one launch; no target twice or also a source."""
        stores = [s[None] for s in (self.table, self._seen, self._counts, self._masks, self.bias_ids, self.biases) if s.numel()]
        kernels.copy_pages([(s, sources, targets) for s in stores])
        self._host[np.asarray(targets, dtype=np.int64)] = self._host[np.asarray(sources, dtype=np.int64)]
