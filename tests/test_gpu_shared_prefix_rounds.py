"""Own blocks that end inside a round of the warps that read them (three blocks a round at
head_dim 128, four at 64): some warps have no block in the last round while others still read
the round before.  Many blocks on every SM and many calls, every one of the same bits."""

import pytest
import torch

from tests.test_gpu_shared_prefix import BF, HF, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,Kh,D,dtype,B", [
    (96, 8, 128, HF, 40), (320, 8, 128, BF, 17), (36, 3, 128, HF, 40), (20, 4, 128, HF, 90),
    (8, 8, 128, BF, 60), (96, 8, 64, BF, 60), (36, 3, 64, HF, 90)])
@pytest.mark.parametrize("group", [False, True])
def test_rounds_with_warps_without_a_block(H, Kh, D, dtype, B, group):
    shared = 5 if group else 0
    lens = [16 * shared + 1 + (37 * i) % 900 for i in range(B)]
    b = Batch(H, Kh, D, dtype, lens, [(range(0, B, 2), shared)] if group else [], seed=B + D,
              poison=True, spread=8.0 if H != 20 else 0.3)
    b.row_blocks = [n + (i % 7) * 4 for i, n in enumerate(b.row_blocks)]
    for full in (False, True):
        plan = b.plan(full_grid=full)
        first = b.run(plan)
        # fp16 results below 2^-14 are held in steps of 2^-24, which the tolerance of the
        # comparison does not count: such results are compared by their bits alone
        ref, tol = b.reference()
        err = (first.view(B, H, D).double() - ref).abs()
        assert (err <= tol + (2.0 ** -25 if dtype == HF else 0.0)).all()
        for _ in range(100):
            assert torch.equal(b.run(plan), first)
