"""Sampled decoding and shared-prefix attention as the model and the engine run them."""

import numpy as np
import pytest
import torch

from agentserve_b200 import (B200Engine, B200LlamaModel, DeviceBlockAllocator, ModelConfig, Request,
                             SamplingParams, UniformStream)
from oracle import sampling as OS

pytestmark = pytest.mark.gpu
CFG = ModelConfig(hidden_dim=512, n_heads=8, n_kv_heads=2, n_layers=2, vocab_size=1000,
                  max_seq_len=2048, intermediate_size=256, rope_theta=10000.0)
WIDE = ModelConfig(hidden_dim=512, n_heads=8, n_kv_heads=2, n_layers=2, vocab_size=5000,
                   max_seq_len=2048, intermediate_size=256, rope_theta=10000.0)


def make_model(dtype, cfg=CFG, seed=0):
    torch.manual_seed(seed)
    m = B200LlamaModel(cfg, dtype=dtype, device="cuda", reference_compat=False)
    with torch.no_grad():
        for p in m.parameters():
            if p.dim() > 1:
                p.normal_(0, 0.05)
        m.lm_head.weight.normal_(0, 0.2)
    return m


def sessions(n, prefix=400, seed=1, max_tokens=12, **kw):
    g = np.random.default_rng(seed)
    shared = g.integers(3, CFG.vocab_size, prefix).tolist()
    return [Request(prompt=f"s{i}", token_ids=shared + g.integers(3, CFG.vocab_size, 5 + 7 * i).tolist(),
                    max_tokens=max_tokens + i % 5, request_id=f"req{i}", **kw) for i in range(n)]


def run(model, requests, cap=8, **kw):
    eng = B200Engine(model.config, model=model, max_batch_size=cap, num_cache_blocks=1500,
                     eos_token_id=-1, use_combined_batching=True, **kw)
    # the first request alone, so the others hit its prefix in the cache
    eng.generate(requests[:1])
    done = eng.generate(requests[1:])
    return {r.request_id: r.output_token_ids for r in done}, eng


def test_engine_tokens_with_shared_prefix_attention():
    """fp32: the same greedy tokens as the per-request attention (its logits differ by
    rounding alone), through graphs whose groups change as requests come and go."""
    model = make_model(torch.float32)
    model.shared_prefix_min_saved = 1
    want, _ = run(model, sessions(13))
    got, eng = run(model, sessions(13), shared_prefix_attention=True)
    assert got == want
    assert eng.metrics.prefix_cache_hits >= 12
    assert any(key[-1] for key in model._graphs), "no step shared blocks"
    model.release_decode_graphs()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step_logits_with_shared_prefix_attention(dtype):
    """One decode step of requests that share blocks, graphed and eager, against the same
    step without sharing.  fp32: sums in another order, 2e-4 as for the model's other
    paths.  bf16: two roundings to bf16 per layer differ, so the two runs are no further
    from each other than each may be from fp32: 2e-2 of the largest logit."""
    model = make_model(dtype)
    alloc = DeviceBlockAllocator(400, num_layers=2, num_kv_heads=2, head_dim=64, dtype=dtype,
                                 device="cuda", max_seqs=16, max_blocks_per_seq=64)
    g = np.random.default_rng(0)
    shared = g.integers(0, 1000, 320).tolist()
    prompts = [shared + g.integers(0, 1000, n).tolist() for n in (3, 40, 17, 90)]
    prompts.append(g.integers(0, 1000, 77).tolist())
    rids = [f"r{i}" for i in range(5)]
    alloc.allocate("r0", 30)
    model.prefill_paged_greedy(prompts[:1], [0], alloc, rids[:1])
    for i in (1, 2, 3):
        alloc.share_blocks(rids[i], alloc.blocks_for("r0")[:20])
        alloc.allocate(rids[i], 10)
    alloc.allocate("r4", 10)
    model.prefill_paged_greedy(prompts[1:], [320, 320, 320, 0], alloc, rids[1:])
    lens = [len(p) for p in prompts]
    model.shared_prefix_min_saved = 1
    ref, _ = model.forward_decode_paged([1, 2, 3, 4, 5], lens, lens, alloc, rids)
    model.shared_prefix_decode = True
    got, _ = model.forward_decode_paged([1, 2, 3, 4, 5], lens, lens, alloc, rids)
    model.decode_graphs = False
    eager, _ = model.forward_decode_paged([1, 2, 3, 4, 5], lens, lens, alloc, rids)
    model.decode_graphs = True
    tol = 2e-4 if dtype == torch.float32 else 2e-2 * ref.float().abs().max().item()
    for x in (got, eager):
        assert (x.float() - ref.float()).abs().max().item() <= tol
    # another batch of the same size through the same graph: the plan follows
    order = [4, 2, 0, 1, 3]
    again, _ = model.forward_decode_paged([5, 3, 1, 2, 4], [lens[i] for i in order],
                                          [lens[i] for i in order], alloc,
                                          [rids[i] for i in order])
    assert (again.float() - ref.float()[order]).abs().max().item() <= tol
    model.release_decode_graphs()


@pytest.mark.parametrize("cfg", [CFG, WIDE])
def test_sampled_step_draws_from_its_logits(cfg):
    """decode_paged_sampled's tokens are the oracle's draws from the step's own logits,
    every request with its own settings."""
    model = make_model(torch.bfloat16, cfg)
    alloc = DeviceBlockAllocator(200, num_layers=2, num_kv_heads=2, head_dim=64,
                                 dtype=torch.bfloat16, device="cuda", max_seqs=16,
                                 max_blocks_per_seq=32)
    g = np.random.default_rng(5)
    # eight requests: the sampled step and the one that gives logits run the same shapes,
    # so their logits have the same bits and every draw must agree
    rids = [f"r{i}" for i in range(8)]
    prompts = [g.integers(0, 1000, 20 + 9 * i).tolist() for i in range(8)]
    for r in rids:
        alloc.allocate(r, 8)
    params = [SamplingParams(0.7), SamplingParams(1.2, top_k=20), SamplingParams(0.9, top_p=0.8),
              SamplingParams(0.0), SamplingParams(1.0, top_k=50, top_p=0.9, min_p=0.02),
              SamplingParams(1.5), SamplingParams(0.6, min_p=0.1), SamplingParams(0.0, top_k=3)]
    stream = UniformStream(3)
    first = model.prefill_paged_sampled(prompts, [0] * 8, alloc, rids, params,
                                        stream(rids, [0] * 8))
    logits = model.forward_prefill_paged(prompts, [0] * 8, alloc, rids).float().cpu().numpy()

    def draws(logits, u):
        return [OS.sample(logits[i], u[i], float(np.float32(p.temperature)), p.top_k,
                          float(np.float32(p.top_p)), float(np.float32(p.min_p)))[0]
                for i, p in enumerate(params)]
    assert first == draws(logits, stream(rids, [0] * 8))
    lens = [len(p) for p in prompts]
    last = first
    for step in range(1, 5):
        u = stream(rids, [step] * 8)
        got = model.decode_paged_sampled(last, lens, alloc, rids, params, u)
        logits, _ = model.forward_decode_paged(last, lens, lens, alloc, rids)
        assert got == draws(logits.float().cpu().numpy(), u)
        model.decode_graphs = False
        eager = model.decode_paged_sampled(last, lens, alloc, rids, params, u)
        model.decode_graphs = True
        assert eager == got
        last, lens = got, [n + 1 for n in lens]
    # a batch of five runs as one of eight rows: the padding rows do not matter
    five = model.decode_paged_sampled(last[:5], lens[:5], alloc, rids[:5], params[:5], u[:5])
    assert len(five) == 5 and five == model.decode_paged_sampled(last, lens, alloc, rids, params,
                                                                 u)[:5]
    model.release_decode_graphs()


def test_engine_sampling_is_reproducible():
    """fp32: tokens depend on the seed, the request and its index, not on the batch cap or
    on speculation; another seed gives others; temperature 0 is greedy."""
    model = make_model(torch.float32)
    kw = dict(temperature=0.9, top_p=0.95, top_k=200, seed=11)
    want, eng = run(model, sessions(9), **kw)
    assert eng.spec_stats["used"] > 0
    got, _ = run(model, sessions(9), cap=3, **kw)
    assert got == want
    eng = B200Engine(model.config, model=model, max_batch_size=8, num_cache_blocks=1500,
                     eos_token_id=-1, use_combined_batching=True, **kw)
    eng.speculative_decode = False
    eng.generate(sessions(9)[:1])
    assert {r.request_id: r.output_token_ids for r in eng.generate(sessions(9)[1:])} == want
    other, _ = run(model, sessions(9), **{**kw, "seed": 12})
    assert other != want
    greedy, _ = run(model, sessions(9))
    zero, _ = run(model, sessions(9, temperature=0.0), per_request_sampling=True)
    assert zero == greedy and greedy != want
    model.release_decode_graphs()


def test_engine_per_request_settings_and_sharing_together():
    """Each request's own settings, sampled steps over shared prefixes: the run equals the
    one without sharing (fp32), and greedy requests in the batch keep their tokens."""
    model = make_model(torch.float32)
    model.shared_prefix_min_saved = 1

    def reqs():
        out = sessions(10, temperature=0.8, top_p=0.9)
        for r in out[::3]:
            r.temperature = 0.0
        out[4].top_k, out[5].min_p = 5, 0.1
        return out
    want, _ = run(model, reqs(), per_request_sampling=True, seed=5)
    got, _ = run(model, reqs(), per_request_sampling=True, seed=5, shared_prefix_attention=True)
    assert got == want
    model.shared_prefix_decode = False
    greedy, _ = run(model, sessions(10))
    for i in (0, 3, 6, 9):
        assert want[f"req{i}"] == greedy[f"req{i}"]
    model.release_decode_graphs()
