"""What the model keeps of a batch's shared blocks between steps (host code)."""

import gc
import weakref

import torch

from agentserve_b200 import B200Engine, B200LlamaModel, DeviceBlockAllocator, ModelConfig

CFG = ModelConfig(hidden_dim=128, n_heads=2, n_kv_heads=1, n_layers=1, vocab_size=50,
                  max_seq_len=512, intermediate_size=64)


def make_model():
    model = B200LlamaModel(CFG, dtype=torch.float32, device="cpu")
    model.shared_prefix_decode = True
    return model


def make_allocator(shared=10, requests=("a", "b", "c")):
    alloc = DeviceBlockAllocator(100, device="cpu", allocate_tensor=False, max_seqs=8,
                                 max_blocks_per_seq=64)
    ids = alloc.allocate(requests[0], shared + 2)
    for r in requests[1:]:
        alloc.share_blocks(r, ids[:shared])
        alloc.allocate(r, 2)
    return alloc


def test_a_dropped_allocator_is_released(monkeypatch):
    """The groups of the last batch keep neither the pool nor, past release_decode_graphs(),
    anything of it."""
    model, alloc = make_model(), make_allocator()
    model.shared_prefix_min_saved = 1
    assert model._sharing(alloc, ["a", "b", "c"]) == ([[0, 1, 2]], [10], [12] * 3)
    gone = weakref.ref(alloc)
    del alloc
    gc.collect()
    assert gone() is None
    other = make_allocator(shared=6)  # of the same epoch and requests
    assert model._sharing(other, ["a", "b", "c"]) == ([[0, 1, 2]], [6], [8] * 3)
    assert model._prefix_groups is not None
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: None)
    model.release_decode_graphs()
    assert model._prefix_groups is None


def test_the_threshold_holds_from_the_next_step(monkeypatch):
    """shared_prefix_min_saved is read at every step, also while the groups are known."""
    model, alloc = make_model(), make_allocator()
    rids = ["a", "b", "c"]
    assert model._sharing(alloc, rids) is None  # 20 block reads saved of 1,920
    calls = []
    find = alloc.shared_prefix_groups
    monkeypatch.setattr(alloc, "shared_prefix_groups", lambda *a: calls.append(a) or find(*a))
    for least, shares in ((20, True), (21, False), (0, True)):
        model.shared_prefix_min_saved = least
        assert (model._sharing(alloc, rids) is not None) == shares
    assert not calls  # from the groups that were found before
    alloc.free("c")
    assert model._sharing(alloc, rids[:2]) == ([[0, 1]], [10], [12] * 2)
    assert len(calls) == 1
    alloc.free("b")
    alloc.allocate("b", 3)
    assert model._sharing(alloc, rids[:2]) is None  # nothing shared, whatever the threshold


def test_an_engines_choice_does_not_reach_another_engine_on_the_model():
    """shared_prefix_attention is the engine's, the model's own setting stays as it was."""
    model, rids = make_model(), ["a", "b", "c"]
    model.shared_prefix_decode = False
    model.shared_prefix_min_saved = 1

    def engine(**kw):
        eng = B200Engine(CFG, model=model, num_cache_blocks=100, **kw)
        ids = eng.allocator.allocate("a", 12)
        for r in rids[1:]:
            eng.allocator.share_blocks(r, ids[:10])
            eng.allocator.allocate(r, 2)
        return eng.allocator
    first = engine(shared_prefix_attention=True)
    assert model._sharing(first, rids) is not None
    assert model.shared_prefix_decode is False
    second = engine()
    assert model._sharing(second, rids) is None
    assert model._sharing(first, rids) is not None
    model.shared_prefix_decode = True  # the model's setting holds for all of them
    assert model._sharing(second, rids) is not None
