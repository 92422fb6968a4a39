"""WFD schedule policy (src/decoding/policy.py:16-59): verify depth T_total,
draft depth T_draft; W = T_total // T_draft tokens in flight at steady state.
`SsdPolicy` decodes greedily; `SampledPolicy` draws every token with a number
its position and the seed decide (single-sequence schedulers). Both are lossless:
the committed tokens are those of sequential decoding with the same sampler."""
from __future__ import annotations

import warnings
from dataclasses import dataclass


@dataclass
class SsdPolicy:
    T_total: int = 8
    T_draft: int = 2
    mode: str = "greedy"
    temperature: float = 1.0
    sample_seed: int = 0

    def __post_init__(self) -> None:
        if self.T_draft < 1 or self.T_total < self.T_draft:
            raise ValueError(f"SsdPolicy: the draft depth must lie in [1, T_total] "
                             f"(T_total={self.T_total}, T_draft={self.T_draft})")
        if self.mode != self._mode():
            raise ValueError(f"Unsupported sampling mode {self.mode!r}: {type(self).__name__} decodes "
                             f"{self._mode()!r} (lossless).")
        if self.T_total % self.T_draft:
            warnings.warn(f"SsdPolicy: T_draft={self.T_draft} does not divide T_total={self.T_total}, so the "
                          "number of tokens in flight varies from tick to tick", stacklevel=2)

    @staticmethod
    def _mode() -> str:
        return "greedy"

    @property
    def steady_state_active_size(self) -> int:
        return self.T_total // self.T_draft

    def make_sampler(self):
        from .acceptance import TokenSampler

        return TokenSampler()


@dataclass
class SampledPolicy(SsdPolicy):
    """Tokens drawn with `sample_seed` (acceptance.SeededSampler): temperature,
    then top_k (0: off), top_p (1: off) and min_p (0: off)."""

    mode: str = "sample"
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0

    def __post_init__(self) -> None:
        super().__post_init__()
        self.make_sampler()  # its checks of the parameters

    @staticmethod
    def _mode() -> str:
        return "sample"

    def make_sampler(self):
        from .acceptance import SeededSampler

        return SeededSampler(self.sample_seed, self.temperature, self.top_k, self.top_p, self.min_p)
