"""Token histories, rules on logits and the choice of a token, row by row with numpy in 64 bits (the oracle of the kernels' tests)."""

import numpy as np


def note(seen, counts, slot, tokens, prompt=0, restart=False):
    """``seen`` truth values ``[slots, V]``, ``counts`` ``[slots, V]``, changed in place."""
    if slot < 0 or slot >= seen.shape[0]:
        return
    if restart:
        seen[slot], counts[slot] = False, 0
    for place, token in enumerate(tokens):
        if 0 <= token < seen.shape[1]:
            seen[slot, token] = True
            counts[slot, token] += place >= prompt


def shaped(x, rule, seen, counts, biases, allowed):
    """A row of logits under a slot's rules, 64 bits.  ``rule``: (repetition, presence, frequency); ``biases``: {id: bias}."""
    x = x.astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore"):
        if rule is not None:
            repetition, presence, frequency = (np.float64(np.float32(v)) for v in rule)
            x = np.where(seen, np.where(x > 0, x / repetition, x * repetition), x)
            x = x - frequency * counts
            x = np.where(counts > 0, x - presence, x)
        for token, bias in (biases or {}).items():
            x[token] = x[token] + np.float64(np.float32(bias))
        if allowed is not None:
            x = np.where(allowed, x, -np.inf)
    return x


def choose(x, temperature, draw, top_k=0, top_p=1.0, min_p=0.0):
    """The token of a row of 32-bit logits."""
    x = np.asarray(x, dtype=np.float32)
    if not (x < np.inf).all() or x.max() == -np.inf:
        return -1
    if not temperature > 0:
        return int(np.argmax(x))
    vocab = x.size
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        inverse = np.float32(1.0) / np.float32(temperature)
        best = x.max()
        k = top_k if 0 < top_k < vocab else vocab
        cut = k < vocab or top_p < 1.0 or min_p > 0.0
        scaled = x * inverse
        d = scaled - best * inverse
        if not cut and abs(best * inverse) < 65536:
            d = (x.astype(np.float64) * np.float64(inverse) - np.float64(best * inverse)).astype(np.float32)
        if not np.isfinite(best * inverse):
            d = np.where(x == best, np.float32(0), -np.float32(np.inf))
    d = d.astype(np.float64)
    order = np.argsort(-d, kind="stable")[:k] if cut else np.arange(vocab)
    weights = np.exp(d[order])
    order, weights = order[weights >= min(min_p, 1.0)], weights[weights >= min(min_p, 1.0)]
    sums = np.cumsum(weights)
    if top_p < 1.0:
        sums = sums[:int(np.searchsorted(sums, sums[-1] * top_p, side="left")) + 1]
    place = int(np.searchsorted(sums, draw * sums[-1], side="right"))
    return int(order[min(place, len(sums) - 1)])
