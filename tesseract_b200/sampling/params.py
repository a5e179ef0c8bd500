"""Per-request generation options, with the reference's names and meanings.

``max_tokens`` (default 128), ``temperature`` (default 1.0; 0 means greedy), ``top_p``
(default 1.0, in (0, 1]), ``seed`` and ``stop`` are the options of the reference's
request type and their validation (src/engine/types.rs:14-37; API defaults
src/api/openai.rs:70-96, 160-167).  ``stop_token_ids`` and ``ignore_eos`` are additions
for a token-ids-in, token-ids-out engine.

Not in the reference either: what a request may say about its next tokens.  Its rules are applied to the logits in this order:
``repetition_penalty`` (divides the positive and multiplies the negative logits of tokens of the prompt and the answer),
``frequency_penalty`` (taken off for every time that the answer has a token), ``presence_penalty`` (taken off once),
``logit_bias`` ({token: bias}, up to 1,024), and then only ``allowed_token_ids`` and what ``grammar`` returns may follow (a callable
that is given the tokens generated so far and returns the ids of those that may come next, or a numpy array of truth values, one a
token of the vocabulary; it is asked on the host in front of every token).  With a temperature above 0 the token is drawn from the ``top_k`` most probable (0: all), of those the ones at least ``min_p``
times as probable as the most probable, of those the fewest that hold ``top_p``.
"""

from __future__ import annotations

import math
from dataclasses import dataclass, field
from typing import Callable, Iterable, Mapping, Optional, Sequence, Tuple

import numpy as np

MAX_BIASES = 1024


def single(value: float) -> float:
    """A number as the kernels have it, in 32 bits; what lies beyond their range is an infinity."""
    with np.errstate(over="ignore", under="ignore"):
        return float(np.float32(value))


@dataclass(frozen=True)
class SamplingParams:
    max_tokens: int = 128
    temperature: float = 1.0
    top_p: float = 1.0
    seed: Optional[int] = None
    stop: Tuple[str, ...] = ()
    stop_token_ids: Tuple[int, ...] = ()
    ignore_eos: bool = False
    top_k: int = 0
    min_p: float = 0.0
    repetition_penalty: float = 1.0
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    logit_bias: Optional[Mapping[int, float]] = None
    allowed_token_ids: Optional[Sequence[int]] = None
    grammar: Optional[Callable[[Sequence[int]], Iterable[int]]] = None

    def __post_init__(self):
        object.__setattr__(self, "stop", tuple([self.stop] if isinstance(self.stop, str) else self.stop))
        object.__setattr__(self, "stop_token_ids", tuple(self.stop_token_ids))
        if self.logit_bias is not None:
            object.__setattr__(self, "logit_bias", dict(self.logit_bias))
        if self.allowed_token_ids is not None:
            object.__setattr__(self, "allowed_token_ids", tuple(self.allowed_token_ids))
        self.validate()
        if self.logit_bias is not None:
            object.__setattr__(self, "logit_bias", {int(token): float(bias) for token, bias in self.logit_bias.items()})
        if self.allowed_token_ids is not None:
            object.__setattr__(self, "allowed_token_ids", tuple(int(token) for token in self.allowed_token_ids))

    def validate(self) -> None:
        if self.max_tokens <= 0:
            raise ValueError("max_tokens must be positive")
        if not math.isfinite(self.temperature) or self.temperature < 0.0:
            raise ValueError("temperature must be finite and non-negative")
        if not math.isfinite(self.top_p) or not 0.0 < self.top_p <= 1.0:
            raise ValueError("top_p must be in (0, 1]")
        if any(s == "" for s in self.stop):
            raise ValueError("stop strings must not be empty")
        if not isinstance(self.top_k, (int, np.integer)) or not 0 <= self.top_k < 2 ** 31:
            raise ValueError("top_k must be a number of tokens (0 for all)")
        if not 0.0 <= self.min_p <= 1.0:
            raise ValueError("min_p must be in [0, 1]")
        if not math.isfinite(single(self.repetition_penalty)) or single(self.repetition_penalty) <= 0.0:
            raise ValueError("repetition_penalty must be finite and positive (in 32 bits)")
        if not math.isfinite(single(self.presence_penalty)) or not math.isfinite(single(self.frequency_penalty)):
            raise ValueError("presence_penalty and frequency_penalty must be finite (in 32 bits)")
        if self.logit_bias is not None:
            if len(self.logit_bias) > MAX_BIASES:
                raise ValueError(f"logit_bias takes up to {MAX_BIASES} tokens")
            for token, bias in self.logit_bias.items():
                if not isinstance(token, (int, np.integer)) or token < 0:
                    raise ValueError("logit_bias names tokens by their ids")
                if math.isnan(bias) or single(bias) == math.inf:
                    raise ValueError("biases must be finite in 32 bits (or -inf, which rules a token out)")
        if self.allowed_token_ids is not None:
            if not self.allowed_token_ids:
                raise ValueError("allowed_token_ids must not be empty")
            if any(not isinstance(t, (int, np.integer)) or t < 0 for t in self.allowed_token_ids):
                raise ValueError("allowed_token_ids names tokens by their ids")
        if self.grammar is not None and not callable(self.grammar):
            raise ValueError("grammar must be callable")

    def check_vocabulary(self, vocab: int) -> None:
        """Raise :class:`ValueError` for a token outside a model's vocabulary."""
        named = [*(self.logit_bias or ()), *(self.allowed_token_ids or ())]
        if named and max(named) >= vocab:
            raise ValueError(f"token {max(named)} is outside the vocabulary of {vocab}")

    @property
    def greedy(self) -> bool:
        return self.temperature == 0.0

    @property
    def penalised(self) -> bool:
        return not (self.repetition_penalty == 1.0 and self.presence_penalty == 0.0 and self.frequency_penalty == 0.0)

    @property
    def ruled(self) -> bool:
        """Whether its logits are changed before a token is chosen."""
        return self.penalised or bool(self.logit_bias) or self.allowed_token_ids is not None or self.grammar is not None

    @property
    def cut(self) -> bool:
        """Whether its tokens are drawn from a part of the distribution."""
        return self.temperature > 0.0 and (self.top_p < 1.0 or self.top_k > 0 or self.min_p > 0.0)


@dataclass(frozen=True)
class TokenChoice:
    """How a step's token for a request is chosen, beyond its temperature and draw: its options, how many tokens its prompt has, and the
    mask words of what its grammar allows in this step."""

    params: SamplingParams
    prompt_tokens: int
    allowed: Optional[np.ndarray] = None

    @staticmethod
    def plain(choice: Optional["TokenChoice"], temperature: float, top_p: float) -> bool:
        """Whether neither rules nor a cut say anything about a row's token: whatever its logits are, it has the token that it has
        beside rows of its kind."""
        params = choice.params if choice is not None else None
        if params is not None and params.ruled:
            return False
        return not (temperature > 0.0 and (top_p < 1.0 or (params is not None and (params.top_k > 0 or params.min_p > 0.0))))

    @classmethod
    def of(cls, params: SamplingParams, prompt_tokens: int) -> Optional["TokenChoice"]:
        return cls(params, prompt_tokens) if params.ruled or params.cut else None
