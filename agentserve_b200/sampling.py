"""Sampling settings of a request and the uniform numbers its tokens are drawn with.

AgentServe samples one request at a time with torch's global generator
(agentserve/engine/sampling.py, engine.py:321, 379-383).  Here a whole batch is sampled
in one launch (ops.sample_tokens) from uniform numbers that are a function of (seed,
request, token index): the numbers do not depend on the batch, on the scheduler, or on
whether a step was queued ahead, and equal logits give equal tokens.  Logits may depend on
the batch in their last bits (its size chooses the projections' kernels, and whether
prefixes are shared the attention's), most in 16-bit types; a draw that lies that close to
the border between two tokens may then differ.
"""

from __future__ import annotations

import hashlib
from dataclasses import dataclass
from typing import Dict, List, Sequence

import numpy as np


@dataclass(frozen=True)
class SamplingParams:
    """temperature <= 1e-6 (or NaN): greedy, and nothing else is read.  Otherwise it is finite,
    top_k a whole number (0 and below: off), top_p in (0, 1] (1: off) and min_p in [0, 1]
    (0: off); other values raise ValueError."""
    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0

    def __post_init__(self):
        if self.greedy:
            return
        if self.temperature == float("inf"):
            raise ValueError("temperature must be finite")
        if not 0.0 < self.top_p <= 1.0:
            raise ValueError(f"top_p must be in (0, 1], got {self.top_p}")
        if not 0.0 <= self.min_p <= 1.0:
            raise ValueError(f"min_p must be in [0, 1], got {self.min_p}")
        try:
            int(self.top_k)
        except (TypeError, ValueError, OverflowError):
            raise ValueError(f"top_k must be a whole number, got {self.top_k!r}") from None

    @property
    def greedy(self) -> bool:
        return not self.temperature > 1e-6


_GREEDY = SamplingParams(temperature=0.0)

# rows of the int32 staging buffer after the decode step's own (tokens, lengths, table rows)
STAGED = 5


def stage(out: np.ndarray, params: Sequence[SamplingParams], u: Sequence[float]) -> None:
    """Writes a batch's settings and numbers into out [5, B] int32: temperature, top_k,
    top_p, min_p and u, the fp32 ones by their bits; rows past the batch are greedy.  Nothing
    else of a greedy request is read."""
    n = len(params)
    params = [_GREEDY if p.greedy else p for p in params]
    f = out.view(np.float32)
    out[:] = 0
    f[0, :n] = [p.temperature for p in params]
    out[1, :n] = [min(max(int(p.top_k), 0), 2 ** 31 - 1) for p in params]
    f[2] = 1.0
    f[2, :n] = [p.top_p for p in params]
    f[3, :n] = [p.min_p for p in params]
    f[4, :n] = u


class UniformStream:
    """u(request, n): the number that the request's n-th output token is drawn with, a
    multiple of 2^-24 in [0, 1).  A 64-bit key per request (a hash of the seed and its
    id) plus n steps of the golden-ratio increment, through Steele, Lea and Flood's
    SplitMix64 finaliser."""

    def __init__(self, seed: int = 0):
        self.seed = int(seed)
        self._keys: Dict[str, int] = {}

    def _key(self, request_id: str) -> int:
        k = self._keys.get(request_id)
        if k is None:
            h = hashlib.blake2b(f"{self.seed}:{request_id}".encode(), digest_size=8)
            k = self._keys[request_id] = int.from_bytes(h.digest(), "little")
        return k

    def forget(self, request_id: str) -> None:
        self._keys.pop(request_id, None)

    def __call__(self, request_ids: Sequence[str], index: Sequence[int]) -> List[float]:
        z = np.array([self._key(r) for r in request_ids], dtype=np.uint64)
        with np.errstate(over="ignore"):
            z += (np.array(index, dtype=np.uint64) + np.uint64(1)) * np.uint64(0x9E3779B97F4A7C15)
            z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
            z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
            z ^= z >> np.uint64(31)
        return ((z >> np.uint64(40)).astype(np.float64) * 2.0 ** -24).tolist()
