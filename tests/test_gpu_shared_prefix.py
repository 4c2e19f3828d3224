"""ops.shared_prefix_decode_attention against plain attention in 64 bits, sequence by
sequence over the whole block table.

Tolerance, element by element, from the arithmetic (A = softmax(s) @ |V|, n keys,
S = the largest sum |q_i k_i| scale of a score):
  fp32 sums: a score is off by at most D S 2^-24, its exponential by that much
  relative plus 2^-22 for the base-2 form, sums over n keys by n 2^-24, and numerator
  and denominator both count: 2 (n + D S + 64) 2^-24 A;
  16-bit types: probabilities are rounded to the type for the product with V, off by
  half a step: eps/2 A; the result once more: eps/2 |out|."""

import numpy as np
import pytest
import torch

from agentserve_b200 import _native as N
from agentserve_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Batch:
    """groups: [(members, shared blocks)]; lens: keys of every row."""

    def __init__(self, H, Kh, D, dtype, lens, groups, seed=0, extra=0, poison=False, spread=1.5):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.H, self.Kh, self.D, self.dtype = H, Kh, D, dtype
        self.lens_list, B = lens, len(lens)
        self.groups = [list(m) for m, _ in groups]
        self.prefix = [p for _, p in groups]
        shared = [0] * B
        for m, p in groups:
            for b in m:
                shared[b] = p
        self.row_blocks = [max(-(-n // 16), s) for n, s in zip(lens, shared)]
        total = sum(self.prefix) + sum(r - s for r, s in zip(self.row_blocks, shared)) + 3
        ids = np.random.default_rng(seed).permutation(total).tolist()
        table = np.zeros((B, max(self.row_blocks) + extra + 1), dtype=np.int32)
        for m, p in groups:
            blocks = [ids.pop() for _ in range(p)]
            for b in m:
                table[b, :p] = blocks
        for b in range(B):
            for j in range(shared[b], self.row_blocks[b]):
                table[b, j] = ids.pop()
        self.table = torch.from_numpy(table).to(DEV)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.q = (torch.randn(B, H, D, generator=g, device=DEV) * spread).to(dtype)
        self.k = torch.randn(total, 16, Kh, D, generator=g, device=DEV).to(dtype)
        self.v = torch.randn(total, 16, Kh, D, generator=g, device=DEV).to(dtype)
        if poison:  # whatever no sequence holds: other requests' leavings, NaN and inf
            used = torch.zeros(total, 16, dtype=torch.bool, device=DEV)
            for b in range(B):
                for j in range(self.row_blocks[b]):
                    n = min(16, lens[b] - 16 * j)
                    if n > 0:
                        used[table[b, j], :n] = True
            self.k[~used] = float("nan")
            self.v[~used] = float("inf")
        self.scale = D ** -0.5

    def plan(self, **kw):
        return ops.shared_prefix_plan(self.groups, self.prefix, self.row_blocks, self.H, self.Kh,
                                      self.D, self.dtype, DEV, **kw)

    def run(self, plan=None, ws=None, **kw):
        plan = plan or self.plan()
        ws = ops.new_shared_prefix_workspace(plan) if ws is None else ws
        return ops.shared_prefix_decode_attention(self.q, self.k, self.v, self.table, self.lens,
                                                  plan, self.scale, ws, **kw)

    def reference(self):
        """(softmax(s) V, its tolerance) in 64 bits."""
        B, H, Kh, D = len(self.lens_list), self.H, self.Kh, self.D
        ref = torch.zeros(B, H, D, dtype=torch.float64, device=DEV)
        tol = torch.full_like(ref, 1e-30)
        half = torch.finfo(self.dtype).eps / 2
        for b, n in enumerate(self.lens_list):
            if n == 0:
                continue
            pos = torch.arange(n, device=DEV)
            slot = self.table[b].long()[pos // 16] * 16 + pos % 16
            k = self.k.view(-1, Kh, D)[slot].double().repeat_interleave(H // Kh, 1)
            v = self.v.view(-1, Kh, D)[slot].double().repeat_interleave(H // Kh, 1)
            q = self.q[b].double()
            p = torch.softmax(torch.einsum("hd,nhd->hn", q, k) * self.scale, -1)
            S = float(torch.einsum("hd,nhd->hn", q.abs(), k.abs()).max() * self.scale)
            ref[b] = torch.einsum("hn,nhd->hd", p, v)
            A = torch.einsum("hn,nhd->hd", p, v.abs())
            tol[b] = 2 * (n + D * S + 64) * 2.0 ** -24 * A + half * ref[b].abs()
            if self.dtype != torch.float32:
                tol[b] += half * A
        return ref, tol

    def check(self, out, layout=N.AS_LAYOUT_HEAD_MAJOR):
        B = len(self.lens_list)
        if layout == N.AS_LAYOUT_DIM_MAJOR:
            out = out.view(B, self.D, self.H).transpose(1, 2)
        ref, tol = self.reference()
        err = (out.reshape(B, self.H, self.D).double() - ref).abs()
        worst = (err / tol).max().item()
        assert torch.isfinite(out).all()
        assert worst <= 1.0, f"{worst:.3f} of the tolerance"
        assert ops.device_status(clear=True) == 0


BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("H,Kh,D,dtype", [
    (32, 8, 64, BF), (32, 8, 128, BF), (24, 8, 128, HF), (32, 32, 64, HF), (16, 1, 128, BF),
    (40, 8, 64, BF), (64, 8, 128, HF), (36, 2, 64, BF), (32, 8, 64, FP), (4, 2, 16, FP),
    (6, 2, 80, BF), (6, 3, 256, HF), (5, 5, 33, FP), (48, 1, 128, FP)])
@pytest.mark.parametrize("case", ["one", "several", "ragged"])
def test_against_64_bits(H, Kh, D, dtype, case):
    """Geometries on every path; one group, several with rows alone, odd lengths."""
    if case == "one":
        lens, groups = [161, 163, 170, 200], [([0, 1, 2, 3], 10)]
    elif case == "several":
        lens = [700, 33, 64, 1, 500, 97, 705, 96, 300, 641]
        groups = [([0, 6, 9], 40), ([2, 5, 7], 4), ([4, 8], 17)]
    else:  # a row that ends with its group's blocks, one token more, one alone of length 1
        lens, groups = [48, 49, 64, 65, 1, 47], [([0, 1, 2, 3], 3)]
    b = Batch(H, Kh, D, dtype, lens, groups, seed=D)
    b.check(b.run())


@pytest.mark.parametrize("dtype,D", [(BF, 64), (HF, 128), (FP, 64), (BF, 128)])
@pytest.mark.parametrize("n,blocks", [(2, 1), (3, 7), (8, 8), (9, 9), (32, 33), (33, 130),
                                      (70, 65), (129, 16)])
def test_group_sizes_and_prefix_lengths(dtype, D, n, blocks):
    """Rows below, at and above a tile's; shared blocks that end inside a key tile."""
    lens = [16 * blocks + 1 + (7 * i) % 40 for i in range(n)]
    b = Batch(32, 8, D, dtype, lens, [(range(n), blocks)], seed=n + blocks)
    b.check(b.run())


@pytest.mark.parametrize("dtype,D", [(BF, 64), (HF, 128), (FP, 64)])
def test_long_prefix_few_rows(dtype, D):
    """A long shared part split over the GPU, and long own parts split too."""
    b = Batch(32, 8, D, dtype, [6000, 6011, 9000, 4001], [([0, 1, 2], 374)], seed=3)
    b.check(b.run())


@pytest.mark.parametrize("dtype,D", [(BF, 64), (BF, 128), (HF, 64), (FP, 64), (FP, 16)])
def test_empty_short_and_poisoned(dtype, D):
    """Rows of length 0, rows shorter than their group's blocks (attended alone), and NaN
    and infinity in every pool row that no sequence holds."""
    lens = [0, 100, 320, 331, 40, 0, 17, 335]
    b = Batch(8, 4, D, dtype, lens, [([1, 2, 3, 4, 7], 20), ([0, 6], 1)], seed=8, poison=True)
    out = b.run()
    assert (out[0] == 0).all() and (out[5] == 0).all()
    b.check(out)


def test_nobody_shares():
    b = Batch(32, 8, 64, BF, [1, 100, 1000, 5000], [], seed=5)
    b.check(b.run())
    one = Batch(32, 8, 64, BF, [900], [([0], 20)], seed=6)  # a group of one
    one.check(one.run())


@pytest.mark.parametrize("dtype", [BF, FP])
def test_layouts_strides_and_wide_tables(dtype):
    """The reference's dim-major output, q as columns of a wider row, table rows longer
    than needed and strided."""
    b = Batch(32, 8, 64, dtype, [400, 410, 30, 401], [([0, 1, 3], 24)], seed=4, extra=60)
    b.check(b.run(out_layout=N.AS_LAYOUT_DIM_MAJOR), N.AS_LAYOUT_DIM_MAJOR)
    wide = torch.zeros(4, 48 * 64, dtype=dtype, device=DEV)
    wide[:, 512:512 + 2048] = b.q.view(4, -1)
    b.q = wide[:, 512:512 + 2048].view(4, 32, 64)
    rows = torch.zeros(4, 200, dtype=torch.int32, device=DEV)
    rows[:, :b.table.shape[1]] = b.table
    b.table = rows[:, :b.table.shape[1]]
    b.check(b.run())


@pytest.mark.parametrize("dtype", [BF, FP])
def test_large_scores_and_equal_keys(dtype):
    """Scores in the hundreds (a few keys take everything), and all keys equal."""
    b = Batch(32, 8, 64, dtype, [200, 260, 199], [([0, 1, 2], 12)], seed=14, spread=60.0)
    b.check(b.run())
    b = Batch(32, 8, 64, dtype, [200, 260, 199], [([0, 1, 2], 12)], seed=15)
    b.k.copy_(b.k[:1, :1].expand_as(b.k).clone())
    b.check(b.run())


@pytest.mark.parametrize("dtype", [BF, FP])
def test_repeated_calls_and_workspace(dtype):
    """One workspace over many calls and plans of one batch size; same bits each time;
    the counters at its front are left at zero."""
    a = Batch(32, 8, 64, dtype, [3000, 2990, 2500, 90], [([0, 1, 2], 150)], seed=1)
    c = Batch(32, 8, 64, dtype, [64, 5000, 300, 310], [([2, 3], 10)], seed=2)
    ws = ops.new_shared_prefix_workspace(a.plan())
    first = a.run(ws=ws).clone()
    for _ in range(3):
        c.check(c.run(ws=ws))
        assert torch.equal(a.run(ws=ws), first)
    a.check(first)
    assert int(ws[:4 * 32 * 4].view(torch.int32).abs().sum()) == 0


def test_lengths_grow_under_one_plan():
    """The plan holds while the rows decode: only lengths change."""
    b = Batch(32, 8, 64, BF, [330, 337, 350, 500], [([0, 1, 2], 20)], seed=7)
    plan = b.plan()
    ws = ops.new_shared_prefix_workspace(plan)
    for step in range(0, 14, 2):
        b.lens_list = [320 + step // 2, 324 + step, 337 + step, 1 + 30 * step]
        b.lens = torch.tensor(b.lens_list, dtype=torch.int32, device=DEV)
        b.check(b.run(plan, ws))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_captured_launch_follows_a_new_plan(dtype):
    """full_grid: one captured call, replayed under plans with other groups."""
    b = Batch(32, 8, 64, dtype, [800, 810, 820, 400, 410, 90],
              [([0, 1, 2], 48), ([3, 4], 20)], seed=11)
    plan = b.plan(full_grid=True)
    ws = ops.new_shared_prefix_workspace(plan)
    out = torch.empty(6, 32 * 64, dtype=dtype, device=DEV)
    b.run(plan, ws, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run(plan, ws, out=out)
    for groups, prefix in ((b.groups, b.prefix), ([[1, 2]], [48]), ([], []),
                           ([[0, 1, 2], [4, 3]], [30, 3])):
        plan.load(groups, prefix, b.row_blocks)
        out.zero_()
        graph.replay()
        b.check(out)


def test_two_streams_with_workspaces_of_their_own():
    b = Batch(32, 8, 64, BF, [2000 + i for i in range(24)], [(range(24), 120)], seed=12)
    c = Batch(32, 8, 128, BF, [1500 + i for i in range(16)], [(range(16), 90)], seed=13)
    pb, pc = b.plan(), c.plan()
    wb, wc = ops.new_shared_prefix_workspace(pb), ops.new_shared_prefix_workspace(pc)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(5):
        outs.append((b, b.run(pb, wb)))
        with torch.cuda.stream(side):
            outs.append((c, c.run(pc, wc)))
    torch.cuda.current_stream().wait_stream(side)
    for who, out in outs:
        who.check(out)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_follows_the_step_that_wrote_the_new_token(dtype):
    """As the decode step uses it: rotate and write the new token, then attend, with no
    synchronisation between; equal to paged_decode_attention up to rounding."""
    b = Batch(32, 8, 64, dtype, [513, 520, 530, 700], [([0, 1, 2, 3], 32)], seed=16)
    g = torch.Generator(device=DEV).manual_seed(1)
    table = torch.randn(1024, 64, generator=g, device=DEV)
    plan = b.plan()
    ws = ops.new_shared_prefix_workspace(plan)
    pos = (b.lens - 1).long()
    slots = b.table.gather(1, (pos // 16).view(-1, 1)).view(-1).long() * 16 + pos % 16
    qkv = torch.randn(4, 48, 64, generator=g, device=DEV).to(dtype)
    out = None
    for _ in range(20):
        t = qkv.clone()
        ops.rope_reshape_and_cache(t[:, :32], t[:, 32:40], t[:, 40:], pos, slots, table, b.k, b.v)
        out = ops.shared_prefix_decode_attention(t[:, :32], b.k, b.v, b.table, b.lens, plan,
                                                 b.scale, ws)
        b.q = t[:, :32].clone()
    b.check(out)


def test_bad_block_ids_are_flagged_and_skipped():
    """Ids outside the pool set status bit 1; nothing out of range is read, and rows
    with good ids keep their results."""
    for dtype in (BF, FP):
        b = Batch(32, 8, 64, dtype, [200, 210, 90, 95], [([0, 1], 12)], seed=17)
        good = b.run().clone()
        ops.device_status(clear=True)
        b.table[2, 3] = b.k.shape[0]
        b.table[3, 0] = -1
        out = b.run()
        assert ops.device_status(clear=True) & 1
        assert torch.equal(out[:2], good[:2])
        b.table[:2, 5] = 1 << 30  # in the shared part
        b.run()
        assert ops.device_status(clear=True) & 1
        # a sequence longer than its table row: flagged, cut to the row
        b = Batch(32, 8, 64, dtype, [200, 210, 90, 95], [([0, 1], 12)], seed=17)
        b.lens[2] = 16 * b.table.shape[1] + 1
        b.run()
        assert ops.device_status(clear=True) & 16
