"""What a request may ask of the sampler.  lucciola's request carries max_new_tokens only
(include/async_engine.h:15-20) and always takes the largest logit; temperature and the filters are added here."""
from __future__ import annotations

from dataclasses import dataclass


@dataclass
class SamplingParams:
    max_new_tokens: int = 16
    temperature: float = 0.0          # 0: greedy
    seed: int = 0                     # stream of random numbers of a request with temperature > 0
    ignore_eos: bool = False          # keep generating past an end-of-sequence token
    # Filters of a draw (temperature > 0), in this order; see ops.sample:
    top_k: int = 0                    # keep this many of the likeliest tokens (0: all)
    top_p: float = 1.0                # of those, the likeliest that make up this part of their probability (1: all)
    min_p: float = 0.0                # of those, the ones at least this many times as likely as the likeliest (0: all)

    def validate(self) -> None:
        if self.max_new_tokens <= 0:
            raise ValueError(f"max_new_tokens must be positive, got {self.max_new_tokens}")
        if self.temperature < 0:
            raise ValueError(f"temperature must not be negative, got {self.temperature}")
        if not 0 <= self.top_k < 2 ** 31:
            raise ValueError(f"top_k must be a number of tokens (0: all), got {self.top_k}")
        if not 0 < self.top_p <= 1:
            raise ValueError(f"top_p must be in (0, 1], got {self.top_p}")
        if not 0 <= self.min_p <= 1:
            raise ValueError(f"min_p must be in [0, 1], got {self.min_p}")

    @property
    def filtered(self) -> bool:
        """Whether a draw of this request leaves tokens out."""
        return self.temperature > 0 and (self.top_k > 0 or self.top_p < 1 or self.min_p > 0)
