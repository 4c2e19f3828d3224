"""ops.sample_tokens against the 64-bit oracle, row by row.

Tokens must be equal: the kernel's weights are 64-bit and its sums exact, so a token can
differ only where u lies within ~1e-12 of a border between two tokens, which the seeds
here do not hit; borders that a test puts there on purpose are exact in both.
Log-probabilities: fp32 rounding of the result (2^-24 relative) and of nothing else; the
64-bit values behind both sides agree to 1e-11, so rtol is 2^-24 + 1e-11 and the
absolute part 1e-11."""

import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from agentserve_b200 import ops
from oracle import sampling as OS

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rows_of(values, dtype):
    return torch.tensor(values, dtype=dtype, device=DEV)


def check(logits, u, T, k=None, p=None, mp=None):
    B = logits.shape[0]
    lp = torch.full((B,), 7.0, device=DEV)
    tok = ops.sample_tokens(logits, rows_of(u, torch.float32), rows_of(T, torch.float32),
                            None if k is None else rows_of(k, torch.int32),
                            None if p is None else rows_of(p, torch.float32),
                            None if mp is None else rows_of(mp, torch.float32), logprobs=lp)
    host = logits.float().cpu().numpy()
    want, want_lp = [], []
    for r in range(B):
        t, l = OS.sample(host[r], float(np.float32(u[r])), float(np.float32(T[r])),
                         0 if k is None else k[r], 1.0 if p is None else float(np.float32(p[r])),
                         0.0 if mp is None else float(np.float32(mp[r])))
        want.append(t)
        want_lp.append(l)
    assert tok.tolist() == want
    np.testing.assert_allclose(lp.cpu().numpy(), np.array(want_lp), rtol=2.0 ** -24 + 1e-11,
                               atol=1e-11)
    return tok


def random_logits(B, V, seed, dtype, spread=2.2):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(B, V, generator=g, device=DEV) * spread
    few = min(V, 20)
    x.scatter_add_(1, torch.randint(0, V, (B, few), generator=g, device=DEV),
                   10.0 * torch.rand(B, few, generator=g, device=DEV))
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (5, 33), (4, 256), (3, 1000), (2, 8193), (9, 32003),
                                 (2, 128256)])
def test_sample_mixed_settings(B, V, dtype):
    """Every filter alone and together, odd sizes, one row to several."""
    g = torch.Generator().manual_seed(B * 1000 + V)
    for trial in range(3):
        T = [float(x) for x in 0.2 + 1.5 * torch.rand(B, generator=g)]
        k = [int(x) for x in torch.randint(0, 60, (B,), generator=g)]
        p = [float(x) for x in 0.3 + 0.9 * torch.rand(B, generator=g)]
        mp = [max(0.0, float(x)) for x in 0.3 * torch.rand(B, generator=g) - 0.1]
        u = torch.rand(B, generator=g).tolist()
        x = random_logits(B, V, trial + V, dtype)
        check(x, u, T)
        check(x, u, T, k=k)
        check(x, u, T, mp=mp)
        check(x, u, T, p=p)
        check(x, u, T, k=k, p=p, mp=mp)


def test_sample_greedy_rows_match_greedy_argmax():
    """Temperature 0 (and NaN), top_k 1 and top_p 0 give the greedy token."""
    x = random_logits(6, 5003, 1, torch.bfloat16)
    x[2, 7] = x[2, 4000] = 60.0  # a tie at the maximum: the first index
    T = [0.0, 1e-6, float("nan"), 1.0, 1.0, 1.0]
    tok = ops.sample_tokens(x, rows_of([0.9] * 6, torch.float32), rows_of(T, torch.float32),
                            rows_of([0, 0, 0, 1, 0, 0], torch.int32),
                            rows_of([1.0, 1.0, 1.0, 1.0, 0.0, 1.0], torch.float32),
                            rows_of([0.0, 0.0, 0.0, 0.0, 0.0, 1.5], torch.float32))
    assert tok.tolist() == ops.greedy_argmax(x).tolist()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sample_ties_at_every_border(dtype):
    """All logits equal: every sum is a whole number, so each border is met exactly."""
    V = 1000
    x = torch.full((6, V), 3.0, device=DEV, dtype=dtype)
    check(x, [0.0, 0.5, 0.25, 0.999, 0.5, 0.75], [0.7] * 6)
    # top-k keeps the first k by index; top-p half of them; u on and between borders
    check(x, [0.0, 0.5, 0.25, 0.999, 0.5, 0.75], [0.7] * 6, k=[8, 8, 8, 8, 1000, 4],
          p=[1.0, 0.5, 0.5, 0.5, 0.5, 1.0], mp=[0.0, 0.0, 1.0, 0.0, 0.0, 1.0])


def test_sample_tie_quota_across_runs():
    """Ties at the cut spread over the whole row: the lowest indexes are kept."""
    V = 20011
    x = torch.full((4, V), -4.0, device=DEV)
    at = torch.arange(3, V, 97, device=DEV)
    x[:, at] = 2.0
    x[:, 19000] = 5.0
    n = len(at)
    for k in (1 + n // 2, 2, n, n + 1, n + 2):
        check(x, [0.1, 0.6, 0.95, 0.9999], [1.3] * 4, k=[k] * 4)
        check(x, [0.1, 0.6, 0.95, 0.9999], [1.3] * 4, k=[k] * 4, p=[0.9] * 4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_sample_masked_and_non_finite_logits(dtype):
    """-inf and the type's lowest value as masks, whole rows masked, NaN, +inf."""
    V = 4099
    x = random_logits(8, V, 5, dtype)
    x[0, 10:] = float("-inf")
    x[1, 1:] = torch.finfo(dtype).min
    x[2, :] = float("-inf")               # nothing left: uniform over the row
    x[3, :] = torch.finfo(dtype).min
    x[4, 17] = float("nan")
    x[5, 4000] = float("inf")
    x[6, :] = float("nan")
    x[7, 5] = torch.finfo(dtype).max
    u = [0.3, 0.999, 0.5, 0.25, 0.7, 0.2, 0.125, 0.4]
    check(x, u, [0.8] * 8)
    check(x, u, [0.8] * 8, k=[50] * 8, p=[0.9] * 8, mp=[0.01] * 8)
    check(x, u, [0.8] * 8, p=[0.75] * 8)


def test_sample_extreme_settings():
    """Temperatures from nearly zero to infinite, filters past the row's size, u at and
    outside its ends."""
    x = random_logits(7, 777, 9, torch.float32)
    T = [1e-3, 1e-5, 50.0, 1e30, float("inf"), 1.0, 1.0]
    check(x, [0.4] * 7, T)
    check(x, [0.4] * 7, T, k=[5, 776, 777, 778, 2 ** 31 - 1, -3, 2], p=[0.999999] * 7,
          mp=[1e-30] * 7)
    check(x, [0.0, 1.0, -1.0, 2.0, 0.99999994, 0.0, 1.0], [0.9] * 7, p=[0.95] * 7)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,V", [(2, 30011), (3, 4096), (200, 2500)])
def test_sample_small_and_large_values(B, V, dtype):
    """Logits all next to zero, on both sides of it, large, and far apart: cuts among
    values of every size."""
    g = torch.Generator(device=DEV).manual_seed(V)
    n = torch.randn(B, V, generator=g, device=DEV)
    u = torch.rand(B, generator=torch.Generator().manual_seed(B)).tolist()
    for x in (n * 1e-3, n * 1e-5, n * 0.02, n * 3e-39, n * 40.0, n.abs() * 200.0, -n.abs() * 300.0,
              -n.abs() * 0.01, torch.where(n > 0, n * 1e-4, n * 8.0),
              torch.where(n > 1.5, 0.0, -500.0) + 0 * n, torch.where(n > 0, 0.0, -0.0)):
        x = x.to(dtype)
        check(x, u, [0.7] * B, p=[0.6] * B)
        check(x, u, [1.1] * B, k=[V // 3] * B, p=[0.97] * B, mp=[0.001] * B)
        check(x, u, [0.05] * B, k=[V // 2] * B)
        if B < 100:
            check(x, u, [60.0] * B, p=[0.5] * B)


def test_sample_u_zero_skips_nothing_of_positive_weight():
    """u = 0 takes the first kept token however unlikely, but none of weight 0."""
    x = torch.tensor([[-60.0, 0.0, 3.0], [-900.0, 0.0, 3.0]], device=DEV)
    tok = check(x, [0.0, 0.0], [1.0, 1.0])
    assert tok.tolist() == [0, 1]


def test_sample_row_strides_and_unaligned_rows():
    """Column slices of a wider buffer whose rows start at odd addresses."""
    big = random_logits(5, 3001, 21, torch.bfloat16)
    check(big[:, 3:2900], [0.1, 0.3, 0.5, 0.7, 0.9], [1.0] * 5, p=[0.9] * 5)
    check(big[::2, 1:], [0.2, 0.5, 0.8], [1.0] * 3, k=[40] * 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,V", [(6, 2049), (3, 30001), (160, 33333)])
def test_sample_rows_from_every_alignment(B, V, dtype):
    """A base at every place within 16 bytes, rows each from another one (odd strides),
    the tokens before and behind the rows larger than any of theirs."""
    for lead in range(128 // torch.finfo(dtype).bits):
        flat = torch.full((lead + B * (V + 2),), 100.0, dtype=dtype, device=DEV)
        x = flat[lead:].view(B, V + 2)[:, :V]
        x.copy_(random_logits(B, V, lead, dtype))
        n = min(B, 8)
        g = torch.Generator().manual_seed(lead)
        u = torch.rand(B, generator=g).tolist()
        u[0], u[1] = 0.0, 1.0 - 2.0 ** -24
        check(x, u, [0.9] * B, k=[50, 0] * (B // 2) + [7] * (B % 2), p=[0.95] * B)
        check(x[:n], u[:n], [1.3] * n)
        assert torch.equal(ops.sample_tokens(x, rows_of(u, torch.float32),
                                             rows_of([0.0] * B, torch.float32)),
                           x.float().argmax(1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_sample_row_does_not_depend_on_its_batch(dtype):
    """Rows in batches of every cluster size: the sums are exact, so tokens and
    log-probabilities are the same bits."""
    x = random_logits(160, 70001, 5, dtype)
    g = torch.Generator(device=DEV).manual_seed(9)
    u = torch.rand(160, generator=g, device=DEV)
    T = 0.3 + torch.rand(160, generator=g, device=DEV)
    k = torch.randint(0, 400, (160,), generator=g, device=DEV, dtype=torch.int32)
    p = 0.7 + 0.4 * torch.rand(160, generator=g, device=DEV)
    want_lp = torch.empty(160, device=DEV)
    want = ops.sample_tokens(x, u, T, k, p, logprobs=want_lp)
    for n in (1, 7, 16, 17, 33, 34, 36, 71, 72, 75, 148, 149):
        lp = torch.empty(n, device=DEV)
        tok = ops.sample_tokens(x[:n], u[:n], T[:n], k[:n], p[:n], logprobs=lp)
        assert torch.equal(tok, want[:n]) and torch.equal(lp, want_lp[:n]), n


def test_sample_frequencies_follow_the_probabilities():
    """Equally spaced u over one row give every kept token its share: the number of the
    N values that fall in a token's interval is off by less than one at either end."""
    N = 4096
    row = random_logits(1, 300, 33, torch.float32)
    x = row.expand(N, -1).contiguous()
    u = (torch.arange(N, device=DEV, dtype=torch.float32) + 0.5) / N
    full = [torch.full((N,), v, device=DEV) for v in (0.7, 0.95)]
    tok = ops.sample_tokens(x, u, full[0], None, full[1]).cpu().numpy()
    kept, w = OS.kept_tokens(row[0].cpu().numpy(), float(np.float32(0.7)),
                             top_p=float(np.float32(0.95)))
    assert set(tok.tolist()) <= set(kept)
    count = np.bincount(tok, minlength=300)[kept]
    assert np.abs(count - N * np.array(w) / sum(w)).max() < 1.0 + 1e-6


def test_sample_is_the_same_in_a_graph_and_on_another_stream():
    x = random_logits(16, 50021, 3, torch.bfloat16)
    u = torch.rand(16, device=DEV)
    T = torch.full((16,), 0.9, device=DEV)
    p = torch.full((16,), 0.9, device=DEV)
    k = torch.full((16,), 300, device=DEV, dtype=torch.int32)
    want = ops.sample_tokens(x, u, T, k, p).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.sample_tokens(x, u, T, k, p)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample_tokens(x, u, T, k, p, out=out)
    for seed in (1, 2):
        u.copy_(torch.rand(16, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        assert torch.equal(out, ops.sample_tokens(x, u, T, k, p))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("value", [0.0, 1.0, -3.0])
def test_sample_the_largest_vocabulary_of_equal_tokens(dtype, value):
    """2^20 tokens of weight 1, the largest sums there are: u picks index u V of the V kept
    ones (exactly, V a power of two), the first V p of them under top-p."""
    V = 1 << 20
    u = [0.0, 0.25, 0.5 + 2.0 ** -20, 0.7109375, 1.0 - 2.0 ** -20]
    flat = torch.full((3 + len(u) * (V + 1),), 50.0, dtype=dtype, device=DEV)
    x = flat[3:].view(len(u), V + 1)[:, :V]
    x.fill_(value)
    ones = [1.0] * len(u)
    for p, kept in ((1.0, V), (0.5, V // 2), (0.0625, V // 16)):
        lp = torch.empty(len(u), device=DEV)
        tok = ops.sample_tokens(x, rows_of(u, torch.float32), rows_of(ones, torch.float32), None,
                                rows_of([p] * len(u), torch.float32), logprobs=lp)
        assert tok.tolist() == [int(v * kept) for v in u]
        torch.testing.assert_close(lp, torch.full_like(lp, -float(np.log(kept))),
                                   rtol=2.0 ** -24 + 1e-11, atol=0)
    k = rows_of([1000, 1, V, V - 1, 3], torch.int32)
    tok = ops.sample_tokens(x, rows_of(u, torch.float32), rows_of(ones, torch.float32), k)
    assert tok.tolist() == [int(v * n) for v, n in zip(u, k.tolist())]


def test_sample_first_call_of_a_process_is_captured():
    """Nothing that the library sets up on a first call breaks a capture."""
    code = """
import torch
from agentserve_b200 import ops
x = torch.randn(20, 50001, device='cuda').half()
u, T = torch.rand(20, device='cuda'), torch.full((20,), 0.9, device='cuda')
out = torch.empty(20, dtype=torch.int64, device='cuda')
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    ops.sample_tokens(x, u, T, out=out)
graph.replay()
assert torch.equal(out, ops.sample_tokens(x, u, T))
"""
    root = Path(__file__).resolve().parents[1]
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True,
                         timeout=300)
    assert run.returncode == 0, run.stderr
