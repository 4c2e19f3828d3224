"""Shared-prefix attention where it can go wrong beside the arithmetic: waits that run out,
pools and queries off the 16-byte boundaries, captured calls that take turns.

A wait is made to run out without a fault: the limit is cut to 1 ms and the next call's
launches issue none of their loads.  The call must come back, set status bit 4 and leave
its workspace as the next call needs it."""

import pytest
import torch

from agentserve_b200 import _native as N
from agentserve_b200 import ops
from tests.test_gpu_shared_prefix import BF, DEV, FP, HF, Batch

pytestmark = pytest.mark.gpu

WAIT_TIMEOUT_BIT = 4


@pytest.fixture
def short_waits():
    lib = N.load()
    ops.device_status(clear=True)
    prev = lib.as_set_wait_limit_ns(1_000_000)  # 1 ms
    yield lib
    lib.as_set_wait_limit_ns(prev)
    lib.as_debug_starve_next_launch(0)
    ops.device_status(clear=True)


@pytest.mark.parametrize("D,dtype", [(64, BF), (128, HF)])
@pytest.mark.parametrize("n", [4, 40])  # one tile in two halves; two streams of rows
def test_wait_that_runs_out_returns_and_next_call_is_correct(short_waits, D, dtype, n):
    lib = short_waits
    b = Batch(32, 8, D, dtype, [1500 + 7 * i for i in range(n)] + [90, 0],
              [(range(n), 90)], seed=D + n)
    plan = b.plan()
    ws = ops.new_shared_prefix_workspace(plan)
    assert lib.as_debug_starve_next_launch(N.AS_KERNEL_SHARED_PREFIX) == N.AS_OK
    starved = b.run(plan, ws)
    torch.cuda.synchronize()
    assert ops.device_status(clear=True) & WAIT_TIMEOUT_BIT
    # a block whose waits ran out leaves empty parts: every row comes out zero
    assert torch.count_nonzero(starved) == 0
    lib.as_set_wait_limit_ns(0)
    b.check(b.run(plan, ws))


@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_pools_and_queries_off_the_boundaries(dtype):
    """Element-aligned pools and queries: one element into their storage, odd row strides."""
    b = Batch(8, 2, 64, dtype, [700, 690, 701, 33], [([0, 1, 2], 40)], seed=5)

    def shifted(x):
        flat = torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)
        y = flat[1:].view(x.shape)
        y.copy_(x)
        return y

    b.check(b.run())
    wide = torch.zeros(4, 8 * 64 + 1, dtype=dtype, device=DEV)
    wide[:, 1:] = b.q.reshape(4, -1)
    b.q = wide[:, 1:].unflatten(1, (8, 64))
    b.check(b.run())
    b.k, b.v = shifted(b.k), shifted(b.v)
    b.check(b.run())


def test_two_captured_graphs_in_turns_on_one_workspace():
    """Two graphs of one batch size and one workspace, replayed one after the other."""
    a = Batch(32, 8, 64, BF, [900, 910, 925, 40], [([0, 1, 2], 50)], seed=1)
    c = Batch(32, 8, 64, BF, [64, 2000, 1300, 1310], [([2, 3], 70), ([0, 1], 4)], seed=2)
    ws = ops.new_shared_prefix_workspace(a.plan(full_grid=True))
    runs = []
    for b in (a, c):
        plan = b.plan(full_grid=True)
        b.run(plan, ws)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = b.run(plan, ws)
        runs.append((b, graph, out, plan))
    for _ in range(3):
        for b, graph, out, _plan in runs:
            out.zero_()
            graph.replay()
        for b, graph, out, _plan in runs:
            b.check(out)


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128)])
def test_a_key_over_everything_in_each_place(dtype, D):
    """One key whose score stands far above all others, moved through the shared blocks:
    the running maximum rises in every tile and stream, and the output is that key's value."""
    b = Batch(32, 8, D, dtype, [777 + i for i in range(5)], [(range(5), 48)], seed=3)
    k0 = b.k.clone()
    for at in (0, 63, 64, 127, 128, 200, 511, 767):
        b.k.copy_(k0)
        slot = int(b.table[0, at // 16]) * 16 + at % 16
        b.k.view(-1, 8, D)[slot] = 12.0 * b.q[0].view(8, 4, D)[:, 0].sign()
        b.check(b.run())
