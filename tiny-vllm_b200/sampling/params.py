"""Per-request sampling parameters; names, defaults and checks of tinyvllm/request.py:32-75, and the rules on logits
(penalties, biases, allowed tokens), which the reference does not have."""

from __future__ import annotations

import math
from dataclasses import dataclass

_MAX_SEED = (1 << 64) - 1
_MAX_BIASES = 1024
_MIN_FLOAT32, _MAX_FLOAT32 = 2.0**-126, (2.0 - 2.0**-23) * 2.0**127          # the device keeps rules in float32


@dataclass(frozen=True)
class SamplingParams:
    max_new_tokens: int = 64
    temperature: float = 0.0        # 0 = greedy
    ignore_eos: bool = False
    seed: int = 0
    top_k: int = 0                  # 0 = off
    top_p: float = 1.0              # 1 = off
    # rules on the logits, in this order (``ops.kernels.logit_rules`` has the formulas)
    repetition_penalty: float = 1.0          # of tokens in the prompt or the answer; 1 = off
    presence_penalty: float = 0.0            # of tokens in the answer
    frequency_penalty: float = 0.0           # ... times their count
    logit_bias: tuple = ()                   # (token, number) pairs, or a mapping
    allowed_token_ids: tuple | None = None   # None = all

    def __post_init__(self) -> None:
        for name in ("max_new_tokens", "seed", "top_k"):
            value = getattr(self, name)
            if type(value) is not int or value < 0:
                raise ValueError(f"{name} must be a non-negative integer")
        if self.seed > _MAX_SEED:
            raise ValueError("seed must fit in 64 bits")
        if type(self.temperature) not in (int, float):
            raise TypeError("temperature must be a number")
        temperature = float(self.temperature)
        if not math.isfinite(temperature) or temperature < 0.0:
            raise ValueError("temperature must be finite and non-negative")
        object.__setattr__(self, "temperature", temperature)
        if type(self.top_p) not in (int, float):
            raise TypeError("top_p must be a number")
        top_p = float(self.top_p)
        if not math.isfinite(top_p) or not 0.0 < top_p <= 1.0:
            raise ValueError("top_p must be in (0, 1]")
        object.__setattr__(self, "top_p", top_p)
        if type(self.ignore_eos) is not bool:
            raise TypeError("ignore_eos must be bool")
        for name in ("repetition_penalty", "presence_penalty", "frequency_penalty"):
            value = getattr(self, name)
            if type(value) not in (int, float):
                raise TypeError(f"{name} must be a number")
            if not abs(value) <= _MAX_FLOAT32 or (name == "repetition_penalty" and value < _MIN_FLOAT32):
                raise ValueError(f"{name} must be finite" + (" and positive" if name == "repetition_penalty" else "") + " in float32")
            object.__setattr__(self, name, float(value))
        pairs = self.logit_bias.items() if hasattr(self.logit_bias, "items") else self.logit_bias
        pairs = tuple(tuple(pair) for pair in pairs)
        for pair in pairs:
            if len(pair) != 2 or type(pair[0]) is not int or pair[0] < 0 or type(pair[1]) not in (int, float) \
                    or not abs(pair[1]) <= _MAX_FLOAT32:
                raise ValueError("logit_bias holds pairs of a token id and a number that is finite in float32")
        if len(pairs) > _MAX_BIASES:
            raise ValueError(f"logit_bias holds up to {_MAX_BIASES} pairs")
        object.__setattr__(self, "logit_bias", pairs)
        if self.allowed_token_ids is not None:
            allowed = tuple(self.allowed_token_ids)
            if not allowed or any(type(token) is not int or token < 0 for token in allowed):
                raise ValueError("allowed_token_ids holds at least one token id (None allows all)")
            object.__setattr__(self, "allowed_token_ids", allowed)
        # (asked of every request of a step: 0.04 us where the five fields take 0.35)
        object.__setattr__(self, "_has_rules", self.repetition_penalty != 1.0 or self.presence_penalty != 0.0 or self.frequency_penalty != 0.0
                           or bool(self.logit_bias) or self.allowed_token_ids is not None)

    @property
    def greedy(self) -> bool:
        return self.temperature == 0.0

    @property
    def has_rules(self) -> bool:
        """Whether the logits are changed before a token is drawn from them."""
        return self._has_rules
