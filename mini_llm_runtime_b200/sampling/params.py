"""How a request chooses its tokens.

The reference chooses greedily only (``argmax`` at src/mini_llm_runtime/engine.py:222,246;
docs/continuous_batch_engine.md:67 names sampling as missing).  Here a request carries a
temperature (0 selects greedy) and a seed.  Both are written into the request's slot record on the
device when it is admitted (cache/slots.py); the sampling kernel (csrc/sampling.cu) reads them by
slot, draws from softmax(logits / temperature) with a counter-based generator keyed by the seed
and the index of the token being produced, and keeps that index in the record.  A request's tokens
therefore depend neither on what else is in its batch nor on how its prompt was cut.

Beside that a request may carry rules on its logits (sampling/rules.py): penalties for the tokens of its prompt and its output,
and biases.  A repetition penalty r divides the logit of every known token by r where it is positive and multiplies it by r
where it is not; frequency and presence penalties are taken off a generated token's logit, once per occurrence and once.
"""

from __future__ import annotations

import math
from collections.abc import Mapping
from dataclasses import dataclass


_LEAST_FLOAT32, _MOST_FLOAT32 = 2.0 ** -126, (2.0 - 2.0 ** -23) * 2.0 ** 127


@dataclass(frozen=True)
class SamplingParams:
    temperature: float = 0.0
    seed: int = 0
    repetition_penalty: float = 1.0
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    logit_bias: tuple[tuple[int, float], ...] = ()      # (token, what is added), ascending; a mapping is taken too

    def __post_init__(self) -> None:
        if isinstance(self.temperature, bool) or not isinstance(self.temperature, (int, float)) \
                or self.temperature < 0:
            raise ValueError("temperature must be a number >= 0 (0 selects greedy)")
        if isinstance(self.seed, bool) or not isinstance(self.seed, int) or not 0 <= self.seed < (1 << 63):
            raise ValueError("seed must be an integer in [0, 2^63)")
        object.__setattr__(self, "temperature", float(self.temperature))
        for name in ("repetition_penalty", "presence_penalty", "frequency_penalty"):
            value = getattr(self, name)
            if isinstance(value, bool) or not isinstance(value, (int, float)) or not math.isfinite(value):
                raise ValueError(f"{name} must be a finite number")
            object.__setattr__(self, name, float(value))
        if self.repetition_penalty <= 0:
            raise ValueError("repetition_penalty must be > 0 (1 changes nothing)")
        # The device holds them in 32 bits, where less would be 0 (and a logit divided by it infinite) and more infinite.
        if not _LEAST_FLOAT32 <= self.repetition_penalty <= _MOST_FLOAT32 or max(abs(self.presence_penalty),
                                                                                abs(self.frequency_penalty)) > _MOST_FLOAT32:
            raise ValueError("penalties must fit 32 bits")
        pairs = self.logit_bias.items() if isinstance(self.logit_bias, Mapping) else self.logit_bias
        biases = tuple(sorted((token, float(value)) for token, value in pairs))
        if any(isinstance(token, bool) or not isinstance(token, int) or token < 0 for token, _ in biases):
            raise ValueError("logit_bias names tokens by integers >= 0")
        if any(math.isnan(value) or value == math.inf for _, value in biases):
            raise ValueError("a bias must be a number; -inf bans its token")
        if any(math.isfinite(value) and abs(value) > _MOST_FLOAT32 for _, value in biases):
            raise ValueError("biases must fit 32 bits")
        if len({token for token, _ in biases}) != len(biases):
            raise ValueError("logit_bias names a token twice")
        object.__setattr__(self, "logit_bias", biases)

    @property
    def greedy(self) -> bool:
        return self.temperature == 0.0

    @property
    def has_rules(self) -> bool:
        return bool(self.logit_bias) or (self.repetition_penalty, self.presence_penalty, self.frequency_penalty) != (1.0, 0.0, 0.0)


GREEDY = SamplingParams()
