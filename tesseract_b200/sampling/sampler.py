"""Choosing tokens from 32-bit logits.

Greedy and temperature rows are chosen on the device by the package's sampling kernel
(argmax with ties to the lowest id, src/cuda/kernels.rs:803-873; inverse-CDF sampling
with the step's uniform draw).  Rows with ``top_p < 1``, the reference's host sampler (src/engine/sampling.rs:38-75:
weights ``exp(l/T - max)`` in 64-bit, sorted by weight, the shortest prefix holding
``top_p`` of the mass, then the draw scaled by the retained mass), are chosen on the device too, by the kernel that also takes top-k,
min-p and a request's rules on its logits (``kernels.choose_tokens``); ``sample_top_p_host`` is the same on the host, for
vocabularies beyond that kernel's.
"""

from __future__ import annotations

from typing import List, Optional, Sequence

import numpy as np
import torch

from .. import kernels
from .params import TokenChoice


class InvalidLogits(ValueError):
    """Empty or non-finite logits reached the sampler (src/engine/sampling.rs:24-27)."""


def sample_top_p_host(logits: np.ndarray, temperature: float, top_p: float, draw: float) -> int:
    if logits.size == 0 or not np.isfinite(logits).all():
        raise InvalidLogits("sampler received empty or non-finite logits")
    if temperature == 0.0:
        return int(np.argmax(logits))
    scaled = logits.astype(np.float32) * (np.float32(1.0) / np.float32(temperature))
    weights = np.exp((scaled - scaled.max()).astype(np.float64))
    order = np.argsort(-weights, kind="stable")
    sorted_weights = weights[order]
    total = float(sorted_weights.sum())
    if not np.isfinite(total) or total <= 0.0:
        raise InvalidLogits("sampler probability mass is invalid")
    cumulative = np.cumsum(sorted_weights)
    kept = int(np.searchsorted(cumulative, total * top_p, side="left")) + 1
    kept = min(kept, logits.size)
    retained = float(cumulative[kept - 1])
    pick = int(np.searchsorted(cumulative[:kept], draw * retained, side="right"))
    return int(order[min(pick, kept - 1)])


class Sampler:
    def __init__(self, device: torch.device):
        self.device = device

    def sample(self, logits: torch.Tensor, temperatures: Sequence[float], top_ps: Sequence[float],
               draws: Sequence[float]) -> List[int]:
        """One token per logits row."""
        rows = logits.shape[0]
        if rows == 0:
            return []
        if not (len(temperatures) == len(top_ps) == len(draws) == rows):
            raise ValueError("one temperature, top_p and draw per logits row")
        if any(t > 0.0 and p < 1.0 for t, p in zip(temperatures, top_ps)) and logits.shape[1] <= kernels.MAX_CHOICE_VOCAB:
            tokens = self.choose(logits, temperatures, draws, top_ps=top_ps,
                                 as_sampled=[TokenChoice.plain(None, t, p) for t, p in zip(temperatures, top_ps)])
            if min(tokens) < 0:
                raise InvalidLogits("sampler received empty or non-finite logits")
            return tokens
        out = torch.empty(rows, dtype=torch.int32, device=self.device)
        if all(t == 0.0 for t in temperatures):
            kernels.argmax(logits, out)
            return out.cpu().tolist()
        temps = torch.tensor(list(temperatures), dtype=torch.float32).to(self.device, non_blocking=True)
        uniform = torch.tensor(list(draws), dtype=torch.float64).to(self.device, non_blocking=True)
        kernels.sample(logits, temps, uniform, out)
        tokens = out.cpu().tolist()
        nucleus = [i for i in range(rows) if temperatures[i] > 0.0 and top_ps[i] < 1.0]
        if nucleus:
            index = torch.tensor(nucleus, dtype=torch.long, device=self.device)
            host = logits.index_select(0, index).cpu().numpy()
            for k, i in enumerate(nucleus):
                tokens[i] = sample_top_p_host(host[k], temperatures[i], top_ps[i], draws[i])
        return tokens

    def choose(self, logits: torch.Tensor, temperatures: Sequence[float], draws: Sequence[float], *,
               top_ks: Optional[Sequence[int]] = None, top_ps: Optional[Sequence[float]] = None,
               min_ps: Optional[Sequence[float]] = None, rules=None, slots: Optional[Sequence[int]] = None,
               as_sampled: Optional[Sequence[bool]] = None) -> List[int]:
        """One token per logits row by ``kernels.choose_tokens``; -1 for a row that has none."""
        rows = logits.shape[0]
        # (one copy for all that a row brings: its 64-bit numbers, then those of 32)
        wide, narrow = np.empty((3, rows), dtype=np.float64), np.zeros((4, rows + rows % 2), dtype=np.int32)
        wide[0], wide[1], wide[2] = draws, 1.0 if top_ps is None else top_ps, 0.0 if min_ps is None else min_ps
        narrow[0, :rows] = np.asarray(temperatures, dtype=np.float32).view(np.int32)
        narrow[1, :rows] = 0 if top_ks is None else top_ks
        narrow[2, :rows] = -1 if slots is None else slots
        narrow[3, :rows] = 0 if as_sampled is None else as_sampled
        sent = torch.from_numpy(np.concatenate([wide.reshape(-1), narrow.reshape(-1).view(np.float64)])).to(self.device)
        wide, narrow = sent[:3 * rows].view(3, rows), sent[3 * rows:].view(torch.int32).view(4, -1)[:, :rows]
        out = torch.empty(rows, dtype=torch.int32, device=self.device)
        kernels.choose_tokens(logits, narrow[0].view(torch.float32), wide[0], out, top_k=narrow[1], top_p=wide[1], min_p=wide[2],
                              rules=rules, slots=narrow[2] if rules is not None else None,
                              as_sampled=narrow[3] if as_sampled is not None else None)
        return out.cpu().tolist()
