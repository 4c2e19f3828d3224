"""Host side of sampled decoding and of shared-prefix batches: settings, uniform
numbers, staging, and the allocator's grouping."""

import itertools
import random

import numpy as np
import pytest

from agentserve_b200 import (B200Engine, DeviceBlockAllocator, Request, SamplingParams,
                             UniformStream)
from agentserve_b200 import sampling as S
from tests.test_engine_host import FAKE_CFG, E


def test_settings_are_checked():
    for bad in (dict(top_p=0.0), dict(top_p=1.5), dict(min_p=-0.1), dict(min_p=1.1),
                dict(temperature=float("inf")), dict(top_p=float("nan")),
                dict(min_p=float("nan"))):
        with pytest.raises(ValueError):
            SamplingParams(**{"temperature": 0.7, **bad})
    assert SamplingParams(temperature=0.0, top_p=0.0).greedy  # nothing of it is used
    assert not SamplingParams().greedy


def test_uniform_numbers_depend_on_seed_request_and_index_alone():
    a, b = UniformStream(7), UniformStream(7)
    rids = [f"r{i}" for i in range(50)]
    whole = np.array([a(rids, [n] * 50) for n in range(40)])
    assert ((whole >= 0) & (whole < 1)).all()
    assert (whole * 2 ** 24 == np.round(whole * 2 ** 24)).all()
    assert b(["r3", "r9"], [5, 11]) == [whole[5, 3], whole[11, 9]]
    a.forget("r3")
    assert a(["r3"], [5]) == [whole[5, 3]]
    assert UniformStream(8)(["r3"], [5]) != [whole[5, 3]]
    assert len(np.unique(whole)) > 1990  # 2000 draws of 2^24 values
    # mean and variance of 2000 uniform numbers, at five standard deviations
    assert abs(whole.mean() - 0.5) < 5 * (1 / 12 / 2000) ** 0.5
    assert abs(whole.var() - 1 / 12) < 5 * (1 / 180 / 2000) ** 0.5


def test_staged_settings():
    out = np.full((S.STAGED, 4), 9, dtype=np.int32)
    S.stage(out, [SamplingParams(0.5, 7, 0.25, 0.125), SamplingParams(2.0, -1)], [0.5, 0.75])
    f = out.view(np.float32)
    assert f[0].tolist() == [0.5, 2.0, 0.0, 0.0]
    assert out[1].tolist() == [7, 0, 0, 0]
    assert f[2].tolist() == [0.25, 1.0, 1.0, 1.0]
    assert f[3].tolist() == [0.125, 0.0, 0.0, 0.0]
    assert f[4].tolist() == [0.5, 0.75, 0.0, 0.0]


def test_engine_refuses_sampling_without_a_sampling_model():
    class Greedy:
        device, dtype, Kh = "cpu", None, 2
    with pytest.raises(ValueError, match="greedy steps only"):
        B200Engine(None, model=Greedy(), temperature=0.8)
    with pytest.raises(ValueError, match="greedy steps only"):
        B200Engine(None, model=Greedy(), per_request_sampling=True)
    with pytest.raises(ValueError, match="top_p"):
        B200Engine(None, model=Greedy(), temperature=0.8, top_p=0.0)
    with pytest.raises(ValueError, match="shared-prefix"):
        B200Engine(None, model=Greedy(), shared_prefix_attention=True)


def test_bad_settings_of_a_request_raise_when_it_is_submitted():
    """Not in a later step, which other requests share."""
    class Sampled(E.HistoryModelForB200):
        def prefill_paged_sampled(self, *args):
            raise AssertionError("no step runs here")

    engine = B200Engine(FAKE_CFG, model=Sampled(), num_cache_blocks=64, per_request_sampling=True)
    good = Request(prompt="a", token_ids=[1, 2], max_tokens=2, temperature=0.7, top_p=0.9)
    bad = Request(prompt="b", token_ids=[1, 2], max_tokens=2, temperature=0.7, top_p=0.0)
    engine.submit(good)
    with pytest.raises(ValueError, match="top_p"):
        engine.submit(bad)
    with pytest.raises(ValueError, match="top_p"):
        engine.submit_many([bad])
    assert list(engine._incoming) == [good]


def allocator(lists):
    a = DeviceBlockAllocator(4096, device="cpu", allocate_tensor=False, max_seqs=64,
                             max_blocks_per_seq=512)
    for i, blocks in enumerate(lists):
        a._request_blocks[str(i)] = list(blocks)
    return a


def groups_of(lists, **kw):
    g, p = allocator(lists).shared_prefix_groups([str(i) for i in range(len(lists))], **kw)
    return sorted((sorted(x), n) for x, n in zip(g, p))


def test_groups_of_a_batch():
    sys = list(range(10))
    assert groups_of([sys + [20], sys + [21, 22], [50, 51], sys]) == [([0, 1, 3], 10)]
    assert groups_of([[1], [2], []]) == []
    # two sessions with long histories below one short system prompt: the histories
    a, b = sys + list(range(100, 300)), sys + list(range(300, 500))
    assert groups_of([a + [600], a + [601], b + [602], b + [603]]) == [([0, 1], 210), ([2, 3], 210)]
    # many requests on the prompt outweigh one pair's short history
    many = [sys + [700 + i] for i in range(20)]
    pair = [sys + [900, 901] + [950 + i] for i in range(2)]
    assert groups_of(many + pair) == [(list(range(22)), 10)]
    assert groups_of([sys + [20], sys + [21]], min_saved=10) == [([0, 1], 10)]
    assert groups_of([sys + [20], sys + [21]], min_saved=11) == []
    long = list(range(1000, 1700))
    assert groups_of([long + [1], long + [2], long[:300]]) == [([0, 1], 700)]


def test_grouping_saves_most_and_is_valid():
    rng = random.Random(3)
    for _ in range(60):
        ids = itertools.count()
        trunk = [next(ids) for _ in range(rng.randint(0, 6))]
        stems = [trunk + [next(ids) for _ in range(rng.randint(0, 9))] for _ in range(3)]
        lists = []
        for _ in range(rng.randint(2, 9)):
            s = rng.choice(stems + [[]])
            lists.append(s[:rng.randint(0, len(s))] + [next(ids) for _ in range(rng.randint(0, 3))])
        got = groups_of(lists)
        seen = [r for g, _ in got for r in g]
        assert len(seen) == len(set(seen))
        for g, n in got:
            assert len(g) > 1 and n > 0
            assert all(lists[r][:n] == lists[g[0]][:n] and len(lists[r]) >= n for r in g)
        # the best partition, by trying every one along the shared beginnings
        def best(rows):
            out = 0
            for n in {k for r in rows for k in range(1, len(lists[r]) + 1)}:
                for head in {tuple(lists[r][:n]) for r in rows if len(lists[r]) >= n}:
                    g = [r for r in rows if tuple(lists[r][:n]) == head and len(lists[r]) >= n]
                    if len(g) > 1:
                        rest = [r for r in rows if r not in g]
                        out = max(out, (len(g) - 1) * n + best(rest))
            return out
        if len(lists) <= 6:
            assert sum((len(g) - 1) * n for g, n in got) >= best(list(range(len(lists))))


def test_a_deep_chain_of_histories():
    """Every request extends the last one's: quick, and still a valid grouping."""
    lists = [list(range(n + 1)) for n in range(300)]
    got = groups_of(lists)
    assert got and all(len(g) > 1 for g, _ in got)
    for g, n in got:
        assert all(len(lists[r]) >= n for r in g)


def test_groups_follow_the_allocator():
    a = DeviceBlockAllocator(100, device="cpu", allocate_tensor=False, max_seqs=8,
                             max_blocks_per_seq=64)
    ids = a.allocate("a", 12)
    e = a.epoch
    a.share_blocks("b", ids[:10])
    a.allocate("b", 2)
    assert a.epoch > e
    assert a.shared_prefix_groups(["a", "b"]) == ([[0, 1]], [10])
    e = a.epoch
    a.free("b")
    assert a.epoch > e and a.shared_prefix_groups(["a", "b"]) == ([], [])
