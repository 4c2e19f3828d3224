"""Captured shared-prefix launches whose plan is replaced by one that shares more blocks than
the captured table holds.  The tables are views of wider ones, so every read that the
operator could make stays inside an allocation; what lies behind the view are ids outside the
pool, which a read would turn into status bit 1."""

import pytest
import torch

from agentserve_b200 import ops
from tests.test_gpu_shared_prefix import BF, DEV, FP, HF, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,D", [(BF, 64), (HF, 128), (FP, 64), (BF, 80)])
def test_a_replayed_plan_wider_than_its_table_is_flagged_and_right(dtype, D):
    b = Batch(32, 8, D, dtype, [480, 470, 475, 300, 310, 90], [([0, 1, 2], 28), ([3, 4], 17)],
              seed=31)
    width = 30  # blocks: 480 keys
    wide = torch.full((6, 200), 1 << 30, dtype=torch.int32, device=DEV)
    wide[:, :width] = b.table[:, :width]
    b.table = wide[:, :width]
    plan = b.plan(full_grid=True)
    ws = ops.new_shared_prefix_workspace(plan)
    out = torch.empty(6, 32 * D, dtype=dtype, device=DEV)
    b.run(plan, ws, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run(plan, ws, out=out)
    graph.replay()
    b.check(out)
    for groups, prefix in (([[0, 1, 2], [3, 4]], [31, 17]), ([[0, 1, 2]], [180]),
                           ([[4, 5], [0, 3, 2]], [31, 199])):
        plan.load(groups, prefix, [200] * 6)
        out.zero_()
        graph.replay()
        # the rows of the wide group fit in the table and are attended alone
        assert ops.device_status(clear=True) == 16
        b.check(out)
        with pytest.raises(ValueError, match="table holds 30"):
            b.run(plan, ws)
    plan.load(b.groups, b.prefix, b.row_blocks)
    out.zero_()
    graph.replay()
    b.check(out)


@pytest.mark.parametrize("dtype,D", [(BF, 64), (HF, 128), (FP, 64)])
@pytest.mark.parametrize("n", [2 ** 31 - 1, 2 ** 31 - 15, 2 ** 31 - 17, 1 << 30])
def test_lengths_near_the_end_of_32_bits_are_flagged_and_cut(dtype, D, n):
    """A row's length past its table: the row is cut to the table, whatever the length."""
    b = Batch(8, 2, D, dtype, [800, 790, 795, 790], [([0, 1], 30)], seed=32)
    wide = torch.full((4, 300), 1 << 30, dtype=torch.int32, device=DEV)
    wide[:, :50] = b.table[:, :50]
    b.table = wide[:, :50]
    want = b.run()
    b.check(want)
    b.lens[0] = b.lens[2] = 800  # the whole table
    b.table[2, 49] = b.table[1, 49]
    want = b.run().clone()
    assert ops.device_status(clear=True) == 0
    b.lens[0] = b.lens[2] = n
    assert torch.equal(b.run(), want)
    assert ops.device_status(clear=True) == 16
