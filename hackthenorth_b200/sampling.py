"""Settings of sampled generation (``Engine.generate(sampling=...)``).

The reference only decodes greedily (``dryft/engine/kernels/greedy.py:45-60``);
this is what its users would set for drawn tokens.
"""
from __future__ import annotations

import dataclasses


@dataclasses.dataclass(frozen=True)
class Sampling:
    """Temperature (0: greedy), then top-k (0: off), top-p (1: off) and min-p
    (0: off), as ``ops.sample_token`` applies them, and the seed of the uniform
    numbers: the same seed, prompts and settings give the same tokens."""

    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    seed: int = 0

    def __post_init__(self):
        if not 0.0 <= self.temperature < float("inf"):
            raise ValueError("temperature must be 0 or more")
        if not (isinstance(self.top_k, int) and 0 <= self.top_k < 2 ** 31):
            raise ValueError("top_k must be a whole number, 0 or more")
        if not 0.0 < self.top_p <= 1.0:
            raise ValueError("top_p must lie in (0, 1]")
        if not 0.0 <= self.min_p <= 1.0:
            raise ValueError("min_p must lie in [0, 1]")
