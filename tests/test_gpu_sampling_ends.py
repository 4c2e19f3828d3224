"""ops.sample_tokens with u at and above 1: the last kept token of positive weight, also
where that weight is far below the units in which sums are held.

Tokens must equal the 64-bit oracle's.  Weights stay above 1e-300, where the oracle's
log-probability is a normal number's."""

import numpy as np
import pytest
import torch

from agentserve_b200 import ops
from tests.test_gpu_sampling import DEV, check, random_logits

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
ENDS = [1.0, 1.0 + 2.0 ** -23, 2.0, float("inf")]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [2, 33, 1000, 1025, 8193, 70001])
def test_u_of_one_takes_the_last_token_however_unlikely(dtype, V):
    x = random_logits(4, V, V, dtype)
    x[:, V - 1] = torch.tensor([-40.0, -100.0, -200.0, -600.0], device=DEV).to(dtype)
    assert check(x, ENDS, [1.0] * 4).tolist() == [V - 1] * 4
    # one that weighs nothing is passed over (1e4 is over 1000 units of the exponent away)
    x[:, V - 1] = -1e4
    assert max(check(x, ENDS, [1.0] * 4).tolist()) < V - 1
    check(x, ENDS, [0.8] * 4, k=[0, 5, 1, 40], p=[0.9, 1.0, 1.0, 0.99], mp=[0.0, 0.0, 0.0, 1e-3])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [64, 1000, 4097, 70001])
def test_u_of_one_counts_ties_at_the_cut(dtype, V):
    """Top-k ends among equal tokens far below the maximum: the first of them by index are
    kept, so the last kept token is the quota's last."""
    x = torch.full((4, V), -1e4, device=DEV, dtype=dtype)
    at = np.arange(1, V, 3)
    x[:, torch.from_numpy(at).to(DEV)] = -50.0
    top = V // 2 // 3 * 3  # not among them
    x[:, top] = 3.0
    n = len(at)
    for k in (2, 1 + n // 2, n, n + 1, n + 2):
        tok = check(x, ENDS, [1.0, 1.0, 0.5, 1.0], k=[k] * 4)
        last = max(top, int(at[min(k - 1, n) - 1]))
        assert tok.tolist() == [last] * 4, k


@pytest.mark.parametrize("dtype", TYPES)
def test_u_of_one_with_masks_and_non_finite_logits(dtype):
    V = 5003
    x = random_logits(5, V, 3, dtype)
    x[0, 3000:] = float("-inf")
    x[1, 100:] = torch.finfo(dtype).min
    x[2, :] = float("-inf")
    x[3, 4000:] = float("nan")
    x[4, 17] = float("inf")
    u = [1.0] * 5
    assert check(x, u, [0.8] * 5).tolist() == [2999, 99, V - 1, V - 1, 17]
    check(x, u, [0.8] * 5, k=[50] * 5, p=[0.9] * 5)
    check(x, u, [1e3] * 5, p=[0.5] * 5)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("V", [5, 1000, 3001, 30011])
def test_the_smallest_positive_weight_counts_at_both_ends(dtype, V):
    """e^-745 rounds to the smallest number above 0 in 64 bits, e^-745.5 to 0."""
    x = torch.full((4, V), -1e4, device=DEV, dtype=dtype)
    x[:, V // 2] = 0.0
    x[0, 1] = x[1, V - 2] = -745.0
    x[2, 1] = x[3, V - 2] = -745.5
    u = torch.tensor([0.0, 1.0, 0.0, 1.0], device=DEV)
    tok = ops.sample_tokens(x, u, torch.ones(4, device=DEV))
    assert tok.tolist() == [1, V - 2, V // 2, V // 2]
