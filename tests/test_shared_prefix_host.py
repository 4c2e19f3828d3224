"""The shared-prefix plan (host code) and the entry points' refusals, without a GPU."""

import ctypes
import random

import numpy as np
import pytest
import torch

from agentserve_b200 import _native as N
from agentserve_b200 import ops

HEADER = 32
ITEM = 8


@pytest.fixture(scope="module")
def lib():
    if not N.LIB_PATH.exists():
        from agentserve_b200.build import build
        build()
    return N.load()


def plan_of(groups, prefix, rows, H=32, Kh=8, D=64, dtype=torch.bfloat16, **kw):
    return ops.shared_prefix_plan(groups, prefix, rows, H, Kh, D, dtype, "cpu", **kw)


def check_covers(p, groups, prefix, rows):
    """Every (member, head of a KV head, shared block) is in one prefix item, the parts
    that items write are disjoint, in range and those the row's own items join, and every
    row has all its own items."""
    h = p._host.tolist()
    B, H, Kh = h[1:4]
    group = H // Kh
    n_pre, n_own, off_mem, off_pre, off_own = h[6], h[7], h[10], h[11], h[12]
    most_prefix, most_own, tile = h[13], h[14], h[15]
    assert h[16] <= p._host.numel() and off_pre % 4 == 0 and off_own % 4 == 0
    want = {}
    for m, n in zip(groups, prefix):
        if len(m) >= 2 and n > 0:
            for b in m:
                want[b] = (n, set(m))
    own, used = {}, set()
    for i in range(n_own):
        it = h[off_own + ITEM * i: off_own + ITEM * (i + 1)]
        assert it[6] > 0
        own.setdefault(it[0], []).append(it)
    for b in range(B):
        items = sorted(own[b], key=lambda x: x[1])
        assert [x[1] for x in items] == list(range(items[0][6]))
        assert all(x[2:] == items[0][2:] for x in items)
        if b not in want:
            assert items[0][2:4] == [0, 0]
        if items[0][6] > 1:
            mine = set(range(items[0][7], items[0][7] + items[0][6]))
            assert not mine & used and max(mine) < most_own
            used |= mine
    assert not any(h[off_own + ITEM * n_own: h[16]])  # unused items are zero
    seen, parts = {}, {}
    for i in range(n_pre):
        row, first, row0, n_rows, begin, end, part, step = h[off_pre + ITEM * i:
                                                             off_pre + ITEM * (i + 1)]
        assert 0 < n_rows <= tile and 0 <= begin < end
        for r in range(row0, row0 + n_rows):
            b = h[off_mem + first + r // group]
            assert row in want[b][1]
            _, _, shared, splits, part0, apart, _, _ = own[b][0]
            assert shared == want[b][0]
            for index in [part + r // group] + ([part + step + r // group] if step else []):
                assert 0 <= index < most_prefix
                assert (index - part0) % apart == 0 and 0 <= (index - part0) // apart < splits
                assert parts.setdefault((index, r % group), i) == i
            seen.setdefault((b, r % group), []).append((begin, end, 2 if step else 1))
    assert not any(h[off_pre + ITEM * n_pre: off_own])
    assert set(b for b, _ in seen) == set(want)
    for b, (n, _) in want.items():
        for e in range(group):
            spans = sorted(seen[b, e])
            assert sum(x[2] for x in spans) == own[b][0][3] <= 64
            assert spans[0][0] == 0 and spans[-1][1] == n
            assert all(x[1] == y[0] for x, y in zip(spans, spans[1:]))
    return h


@pytest.mark.parametrize("H,Kh,D,dtype", [(32, 8, 64, torch.bfloat16), (24, 8, 128, torch.float16),
                                          (16, 1, 128, torch.bfloat16), (32, 32, 64, torch.float16),
                                          (4, 2, 16, torch.float32), (36, 2, 64, torch.bfloat16)])
def test_plan_covers_every_shared_block_once(lib, H, Kh, D, dtype):
    rng = random.Random(H * 131 + D)
    for trial in range(25):
        B = rng.choice([1, 2, 3, 7, 33, 64, 200, 700])
        rows = list(range(B))
        rng.shuffle(rows)
        groups, prefix = [], []
        while rows and len(groups) < 8:
            n = rng.randint(1, max(1, len(rows)))
            groups.append(rows[:n])
            rows = rows[n:]
            prefix.append(rng.choice([0, 1, 5, 8, 100, 2000]))
            if rng.random() < 0.3:
                break
        blocks = [rng.randint(0, 400) for _ in range(B)]
        for m, n in zip(groups, prefix):
            for b in m:
                blocks[b] += n
        for full in (False, True):
            p = plan_of(groups, prefix, blocks, H, Kh, D, dtype, full_grid=full)
            h = check_covers(p, groups, prefix, blocks)
            assert h[8] >= h[6] and h[9] >= h[7]
            if not full:
                assert h[8:10] == h[6:8]


def test_full_grids_depend_on_the_sizes_alone(lib):
    a = plan_of([[0, 1, 2]], [500], [600] * 3 + [9], full_grid=True)
    b = plan_of([], [], [1] * 4, full_grid=True)
    assert a._host.tolist()[8:10] == b._host.tolist()[8:10]
    assert a.workspace_bytes == b.workspace_bytes
    a.load([], [], [1] * 4)
    assert torch.equal(a.ints, b.ints)


@pytest.mark.parametrize("groups,prefix,rows,text", [
    ([[0, 1], [1, 2]], [1, 1], [4] * 4, "different rows"),
    ([[0, 4]], [1], [4] * 4, "different rows"),
    ([[0, -1]], [1], [4] * 4, "different rows"),
    ([[0, 1]], [5], [4] * 4, "fewer blocks"),
    ([[0, 1]], [-1], [4] * 4, "negative prefix_blocks"),
    ([[0, 1]], [1], [4, 4, -1, 4], "negative row_blocks"),
    ([[0, 1]], [1, 2], [4] * 4, "one prefix_blocks per group"),
])
def test_bad_plans_are_refused(lib, groups, prefix, rows, text):
    with pytest.raises(ValueError, match=text):
        plan_of(groups, prefix, rows)


def test_bad_geometries_are_refused(lib):
    for H, Kh, D in ((30, 8, 64), (32, 8, 257), (0, 8, 64), (32, 0, 64)):
        assert lib.as_shared_prefix_plan_ints(4, H, Kh, D, N.AS_DTYPE_BF16) == 0
        assert lib.as_shared_prefix_workspace_size(4, H, Kh, D, N.AS_DTYPE_BF16) == 0
    assert lib.as_shared_prefix_plan_ints(0, 32, 8, 64, N.AS_DTYPE_BF16) == 0
    with pytest.raises(ValueError):
        plan_of([], [], [])
    with pytest.raises(TypeError):
        plan_of([], [], [1], dtype=torch.float64)
    rows = np.ones(4, dtype=np.int32)
    assert lib.as_shared_prefix_plan(None, 0, None, None, None, 0, rows.ctypes.data, 4, 32, 8, 64,
                                     N.AS_DTYPE_BF16, 0) == N.AS_ERR_INVALID_ARG
    buf = np.zeros(8, dtype=np.int32)
    assert lib.as_shared_prefix_plan(buf.ctypes.data, 8, None, None, None, 0, rows.ctypes.data, 4,
                                     32, 8, 64, N.AS_DTYPE_BF16, 0) == N.AS_ERR_INVALID_ARG
    assert "ints" in N.last_error() and not buf.any()


def test_attention_checks_its_arguments_first(lib):
    p = plan_of([[0, 1]], [3], [4] * 4)
    head = p._host.data_ptr()

    def call(B=4, H=32, Kh=8, D=64, bs=16, NB=100, mb=10, stride=10, qs=2048, ptr=256, ws=256,
             n=1 << 40, scale=0.125, layout=0, dtype=N.AS_DTYPE_BF16, header=head):
        return lib.as_shared_prefix_decode_attention(
            ptr, ptr, qs, ptr, ptr, ptr, stride, ptr, header, ptr, B, H, Kh, D, bs, NB, mb, scale,
            ws, n, layout, dtype, None)
    assert call(dtype=7) == N.AS_ERR_INVALID_ARG and "dtype" in N.last_error()
    assert call(bs=8) == N.AS_ERR_UNSUPPORTED and "block_size" in N.last_error()
    for bad in (dict(B=-1), dict(Kh=5), dict(NB=0), dict(mb=0), dict(stride=9), dict(qs=2047)):
        assert call(**bad) == N.AS_ERR_INVALID_ARG and "bad sizes" in N.last_error()
    for bad in (0.0, -0.5, float("nan"), float("inf")):
        assert call(scale=bad) == N.AS_ERR_INVALID_ARG and "scale" in N.last_error()
    assert call(layout=2) == N.AS_ERR_INVALID_ARG and "out_layout" in N.last_error()
    assert call(ptr=None) == N.AS_ERR_INVALID_ARG and "null pointer" in N.last_error()
    for bad in (dict(B=3), dict(H=16, qs=2048), dict(D=32), dict(dtype=N.AS_DTYPE_F16)):
        assert call(**bad) == N.AS_ERR_INVALID_ARG and "another batch" in N.last_error()
    assert call(mb=2, stride=2) == N.AS_ERR_INVALID_ARG and "table holds 2" in N.last_error()
    assert call(n=p.workspace_bytes - 1) == N.AS_ERR_WORKSPACE
    assert call(ws=None) == N.AS_ERR_WORKSPACE
    assert call(ws=128) == N.AS_ERR_INVALID_ARG and "256-byte" in N.last_error()
    assert call(B=0) == N.AS_OK
    blank = (ctypes.c_int32 * HEADER)()
    assert call(header=ctypes.addressof(blank)) == N.AS_ERR_INVALID_ARG


def test_cpu_tensors_are_refused(lib):
    p = plan_of([], [], [1])
    with pytest.raises(RuntimeError):
        ops.shared_prefix_decode_attention(
            torch.zeros(1, 32, 64), torch.zeros(2, 16, 8, 64), torch.zeros(2, 16, 8, 64),
            torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32), p, 0.125)
