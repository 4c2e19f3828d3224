"""Sampling with temperature, top-k, top-p and min-p from a given uniform number, one
row at a time in 64 bits (agentserve/engine/sampling.py's order of filters; min-p is
this library's addition)."""

from __future__ import annotations

import math

import numpy as np


def sanitize(row: np.ndarray) -> np.ndarray:
    """fp32 upcast and nan_to_num(0, 1e4, -1e4) (sampling.py:46-48)."""
    row = np.asarray(row, dtype=np.float32)
    return np.nan_to_num(row, nan=0.0, posinf=1e4, neginf=-1e4)


def kept_tokens(row: np.ndarray, temperature: float, top_k: int = 0, top_p: float = 1.0,
                min_p: float = 0.0):
    """Indexes of the kept tokens in index order and their weights exp((x - max) / T)."""
    x = sanitize(row).astype(np.float64)
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    if not temperature > 1e-6:
        return [order[0]], [1.0]
    weight = {i: math.exp((x[i] - x[order[0]]) / temperature) for i in order}
    n = top_k if 0 < top_k < len(x) else len(x)
    kept = order[:n]
    if top_p < 1.0:
        total, run, cut = math.fsum(weight[i] for i in kept), 0.0, 0
        for cut, i in enumerate(kept, 1):
            run += weight[i]
            if run >= top_p * total:
                break
        kept = kept[:max(cut, 1)] if top_p > 0 else kept[:1]
    if min_p > 0:
        kept = [i for i in kept if weight[i] >= min_p] or kept[:1]
    kept = sorted(kept)
    return kept, [weight[i] for i in kept]


def sample(row: np.ndarray, u: float, temperature: float, top_k: int = 0, top_p: float = 1.0,
           min_p: float = 0.0):
    """(token, log-probability among the kept tokens)."""
    kept, w = kept_tokens(row, temperature, top_k, top_p, min_p)
    total = math.fsum(w)
    cum = np.cumsum(w)
    at = int(np.searchsorted(cum, max(u, 0.0) * cum[-1], side="right"))
    positive = [i for i, x in enumerate(w) if x > 0]
    at = min(max(at, positive[0]), positive[-1])
    return kept[at], math.log(w[at] / total) if w[at] > 0 else -math.inf
