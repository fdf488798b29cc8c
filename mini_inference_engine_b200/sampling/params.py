"""Sampling options of a request: ``SamplingParams`` of inference_engine/sampling.py:6-10
(``max_tokens``, ``temperature`` with 0 = greedy, ``ignore_eos``) plus ``seed``; the reference
draws from torch's global generator, unseeded, so its sampled runs cannot be repeated.  Beside them, what
the reference does not have: penalties for repeated tokens, biases, a grammar, log-probabilities."""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass


def _single(x) -> float:
    """x as the float32 that the kernels get (beyond their range: infinite)."""
    return ctypes.c_float(x).value


@dataclass
class SamplingParams:
    max_tokens: int = 128
    temperature: float = 0.0        # 0 = greedy
    ignore_eos: bool = False        # keep generating past EOS (fixed-length benchmarks)
    seed: int | None = None         # None = the engine's seed
    # rules on the logits, in this order (see kernels.ops.LogitRules); the temperature comes after them
    repetition_penalty: float = 1.0     # > 0: tokens of the prompt and the answer have their logits divided by it (multiplied below 0)
    presence_penalty: float = 0.0       # taken off the logits of tokens that the answer holds ...
    frequency_penalty: float = 0.0      # ... and this once for every time that it holds them
    logit_bias: dict | None = None      # token id -> what is added to its logit (-inf: a ban)
    grammar: object | None = None       # has allowed(output_ids) -> token ids, or one truth value an entry of the vocabulary (or None: all),
                                        # asked before every token; where it allows nothing (but what logit_bias bans), the request ends
    logprobs: bool = False              # the output's logprobs: of every token, under the rules and before the temperature

    def __post_init__(self):
        if self.temperature < 0:
            raise ValueError(f"temperature must be >= 0, got {self.temperature}")
        # (all of them as float32: 1e300 is infinite there, and 1e-46 is 0)
        if not (_single(self.repetition_penalty) > 0 and math.isfinite(_single(self.repetition_penalty))):
            raise ValueError(f"repetition_penalty must be positive and finite in float32, got {self.repetition_penalty}")
        for name in ("presence_penalty", "frequency_penalty"):
            if not math.isfinite(_single(getattr(self, name))):
                raise ValueError(f"{name} must be finite in float32, got {getattr(self, name)}")
        for t, b in (self.logit_bias or {}).items():
            if int(t) != t or t < 0:
                raise ValueError(f"logit_bias: {t!r} is not a token id")
            if math.isnan(b) or _single(b) == math.inf:
                raise ValueError(f"logit_bias of token {t}: a finite number in float32 or -inf, got {b}")
        if self.grammar is not None and not callable(getattr(self.grammar, "allowed", None)):
            raise ValueError("a grammar has a method allowed(output_ids)")

    def banned(self) -> list:
        """Tokens whose bias leaves them no chance."""
        return [int(t) for t, b in (self.logit_bias or {}).items() if _single(b) == -math.inf]

    @property
    def has_rules(self) -> bool:
        """Whether the token is chosen from other logits than the model's, or its log-probability is asked for."""
        return bool(self.repetition_penalty != 1.0 or self.presence_penalty or self.frequency_penalty or self.logit_bias
                    or self.grammar is not None or self.logprobs)
