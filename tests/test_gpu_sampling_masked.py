"""ops.sample_tokens on rows of which a mask leaves few tokens, fewer than top-k asks for, with
the other cuts among values of every size next to zero."""

import numpy as np
import pytest
import torch

from tests.test_gpu_sampling import DEV, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [1000, 3001, 17001])
@pytest.mark.parametrize("mask", ["-inf", "lowest", "-1e4", "-130"])
def test_top_k_past_the_unmasked_tokens(dtype, V, mask):
    g = np.random.default_rng(V)
    B, left = 3, 240
    x = torch.full((B, V), {"-inf": float("-inf"), "lowest": torch.finfo(dtype).min, "-1e4": -1e4,
                            "-130": -130.0}[mask], dtype=dtype, device=DEV)
    for r in range(B):
        at = torch.from_numpy(g.choice(V, left, replace=False)).to(DEV)
        # a third each: around 1, next to zero on both sides (smaller than 2^-9), and below
        near = g.uniform(-1.0, 1.0, left // 3) * 10.0 ** g.uniform(-9, -3, left // 3)
        v = np.concatenate([g.normal(1.0, 0.1, left // 3), near, g.normal(-2.0, 0.5, left // 3)])
        x[r, at] = torch.from_numpy(g.permutation(v).astype(np.float32)).to(DEV).to(dtype)
    u = g.random(B).tolist()
    u[0] = 1.0 - 2.0 ** -24
    T = [1.0, 0.9, 0.7]
    for k in (left, left + 1, left + 100, V - 1):
        for p in (0.6, 0.8, 0.9, 0.99, 0.999999):
            check(x, u, T, k=[k] * B, p=[p] * B)
        check(x, u, T, k=[k] * B, p=[0.9] * B, mp=[0.3] * B)
        check(x, u, T, k=[k] * B)
