"""Token choice and draft acceptance (src/decoding/acceptance.py:40-58; drawn
tokens: acceptance.py:61-214).

A committed token is argmax of the full-depth logits; a draft is accepted iff
it equals that argmax (lossless top-1), otherwise the argmax is committed
instead. Logits may arrive as a tensor or as a `RowLogits`, which carries the
argmax already computed on the device, so a whole coda union costs one
device->host read.

`SeededSampler` draws tokens instead: position p's token is a function of the
logits there and of u(p), a uniform number that the seed alone decides. A draft
and its verification draw with the same number, so a draft is accepted iff the
full-depth logits draw the same token, and the committed tokens are the ones
sequential decoding with the same seed draws.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch


@dataclass
class RowLogits:
    """One row of coda logits with its device-computed argmax."""

    values: torch.Tensor   # (V,) float32 (device view)
    token: int             # argmax (first index on ties)

    def argmax(self, dim: int = -1):
        return torch.tensor(self.token)


def greedy_sample(logits) -> int:
    if isinstance(logits, RowLogits):
        return logits.token
    if logits.dim() > 1:
        logits = logits.reshape(-1)
    return int(logits.argmax(dim=-1).item())


def greedy_accept(draft_token: int, verify_logits) -> tuple[bool, int]:
    target = greedy_sample(verify_logits)
    return draft_token == target, target


class TokenSampler:
    """The sampler every decode path shares so AR and WFD emit the same
    token for the same (position, logits). Greedy."""

    temperature = 0.0

    def __call__(self, logits, position: int) -> int:
        return greedy_sample(logits)

    def draft(self, logits, position: int):
        return greedy_sample(logits), None

    def verify(self, draft_token: int, draft_probs, verify_logits, position: int) -> tuple[bool, int]:
        return greedy_accept(draft_token, verify_logits)


GREEDY = TokenSampler()


class SeededSampler(TokenSampler):
    """Tokens drawn by ops.sample from the position's logits and u(position).
    top_k 0, top_p 1 and min_p 0 are off; temperature 0 is greedy."""

    _BLOCK = 4096  # positions whose numbers are drawn at once

    def __init__(self, seed: int = 0, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
                 min_p: float = 0.0):
        if not (temperature >= 0.0 and top_k >= 0 and 0.0 < top_p <= 1.0 and 0.0 <= min_p <= 1.0):
            raise ValueError(f"SeededSampler: temperature={temperature} top_k={top_k} top_p={top_p} min_p={min_p} "
                             "(temperature, top_k >= 0; top_p in (0, 1]; min_p in [0, 1])")
        self.seed, self.temperature = int(seed), float(temperature)
        self.top_k, self.top_p, self.min_p = int(top_k), float(top_p), float(min_p)
        self._on_device: dict = {}  # parameters and blocks of u per device

    def uniform(self, position: int) -> float:
        return float(self._block(position // self._BLOCK)[position % self._BLOCK])

    def _block(self, index: int) -> torch.Tensor:
        g = torch.Generator().manual_seed((self.seed * 1000003 + index) % (1 << 63))
        return torch.rand(self._BLOCK, generator=g)

    def _tensors(self, device, index: int):
        have = self._on_device.setdefault(device, {})
        if not have:
            have["temperature"] = torch.tensor([self.temperature], device=device)
            k = min(self.top_k, 2 ** 31 - 1)  # beyond any vocabulary: off
            have["top_k"] = torch.tensor([k], dtype=torch.int32, device=device) if k else None
            have["top_p"] = torch.tensor([self.top_p], device=device) if self.top_p < 1.0 else None
            have["min_p"] = torch.tensor([self.min_p], device=device) if self.min_p else None
        if index not in have:
            have[index] = self._block(index).to(device)
        return {k: have[k] for k in ("temperature", "top_k", "top_p", "min_p")}, have[index]

    def __call__(self, logits, position: int) -> int:
        from . import ops

        row = (logits.values if isinstance(logits, RowLogits) else logits).reshape(1, -1)
        params, u = self._tensors(row.device, position // self._BLOCK)
        at = position % self._BLOCK
        return int(ops.sample(row, u[at: at + 1], **params).item())

    def draft(self, logits, position: int):
        return self(logits, position), None

    def verify(self, draft_token: int, draft_probs, verify_logits, position: int) -> tuple[bool, int]:
        target = self(verify_logits, position)
        return draft_token == target, target
