"""Shared-prefix attention over keys and queries that are NaN: what the formula makes of them
(NaN) comes out, however the row's keys are divided into parts, and rows beside them keep
their bits."""

import pytest
import torch

from agentserve_b200 import ops
from tests.test_gpu_shared_prefix import BF, FP, HF, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,D", [(BF, 64), (HF, 128), (FP, 64)])
@pytest.mark.parametrize("where", ["own", "alone", "shared"])
def test_a_block_of_nan_keys_reaches_the_output(dtype, D, where):
    """Sixteen NaN keys: every score of a block, and so all that one warp (or token group)
    may see of a part, is NaN."""
    b = Batch(8, 2, D, dtype, [5000, 4990, 900, 90], [([0, 1], 40)], seed=21)
    good = b.run().clone()
    row = {"own": 0, "alone": 2, "shared": 0}[where]
    for at in {"own": (40, 41, 42, 150, 312), "alone": (0, 7, 56), "shared": (0, 9, 39)}[where]:
        block = int(b.table[row, at])
        kept = b.k[block].clone()
        b.k[block, :, 1] = float("nan")  # of KV head 1: query heads 4 to 7
        out = b.run().view(4, 8, D)
        b.k[block] = kept
        hit = [0, 1] if where == "shared" else [row]
        for r in range(4):
            assert torch.equal(out[r, :4], good.view(4, 8, D)[r, :4]), (at, r)
            if r in hit:
                assert out[r, 4:].isnan().all(), (at, r)
            else:
                assert torch.equal(out[r], good.view(4, 8, D)[r]), (at, r)
    assert ops.device_status(clear=True) == 0


@pytest.mark.parametrize("dtype,D", [(BF, 64), (HF, 128), (FP, 64)])
def test_a_nan_query_gives_nan(dtype, D):
    """All scores of a head NaN: in a group, alone in one part and alone in several."""
    b = Batch(8, 2, D, dtype, [5000, 4990, 9000, 90, 0], [([0, 1], 40)], seed=22)
    good = b.run().clone().view(5, 8, D)
    b.q[:, 5, 3] = float("nan")
    out = b.run().view(5, 8, D)
    assert out[:4, 5].isnan().all()
    assert (out[4] == 0).all()  # no keys
    keep = [0, 1, 2, 3, 4, 6, 7]
    assert torch.equal(out[:, keep], good[:, keep])
