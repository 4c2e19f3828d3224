"""Cases for the two operators of the sampled decode step over a shared prefix:

* shared-prefix decode attention: one new token per sequence attends over its paged
  K/V; groups of sequences hold the same leading 16-token blocks (a prefix-cache hit
  shares them), and those blocks are read and multiplied once for the whole group;
* sampling with temperature, top-k, top-p and min-p from given uniform numbers.

`run` computes them in elementary torch operations, or, where `own` is set, with the
calls a program makes of agentserve_b200.ops.
"""

import random

import numpy as np
import torch

own = False

BLOCK = 16
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _attn(name, dtype, heads, kv_heads, head_dim, seqs, groups, private, prefix, suffix):
    return {"name": name, "op": "attention", "dtype": dtype, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "seqs": seqs, "groups": groups,
            "private": private, "prefix": prefix, "suffix": suffix}


def _samp(name, dtype, rows, vocab, temperature, top_k, top_p, min_p, mixed=False):
    return {"name": name, "op": "sample", "dtype": dtype, "rows": rows, "vocab": vocab,
            "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "mixed": mixed}


def listed():
    return [
        # four sessions on a 160-token system prompt, first tokens of their answers
        _attn("attn 4 on 160", "bf16", 32, 8, 64, 4, 1, 0, 160, 40),
        # the 64-sequence decode step, all agents on one 4K instruction prompt
        _attn("attn 64 on 4096", "bf16", 32, 8, 64, 64, 1, 0, 4096, 512),
        # several agent kinds in one batch, some requests alone; three heads per KV head
        _attn("attn 61 in 5 groups", "fp16", 24, 8, 128, 61, 5, 9, 2480, 700),
        # the session workload: 64 running, 14,336 shared tokens
        _attn("attn 64 on 14336", "bf16", 32, 8, 64, 64, 1, 0, 14336, 1000),
        # the full-precision path that parity tests run
        _attn("attn 16 fp32", "fp32", 32, 8, 64, 16, 2, 2, 1024, 200),
        # a large replica of the 8B geometry near its longest context
        _attn("attn 256 on 30000", "bf16", 32, 8, 128, 256, 2, 0, 30000, 512),
        # one request alone: latency
        _samp("sample 1", "bf16", 1, 128256, 0.7, 0, 0.95, 0.0),
        # the 64-sequence decode step with every request's own settings, some greedy
        _samp("sample 64 mixed", "bf16", 64, 128256, 0.8, 40, 0.9, 0.05, mixed=True),
        # a large batch on top-p alone
        _samp("sample 256 top-p", "bf16", 256, 128256, 0.8, 0, 0.9, 0.0),
        # logits kept in fp32, min-p alone
        _samp("sample 48 fp32 min-p", "fp32", 48, 128256, 1.0, 0, 1.0, 0.05),
        # a smaller odd vocabulary, top-k alone
        _samp("sample 33 fp16 top-k", "fp16", 33, 32003, 0.9, 50, 1.0, 0.0),
        # the tiny test geometry's vocabulary
        _samp("sample 8 of 256", "fp32", 8, 256, 1.0, 20, 0.9, 0.0),
    ]


def _between(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    if rng.random() < 0.5:
        heads, kv_heads, head_dim = rng.choice(
            [(32, 8, 64), (24, 8, 128), (32, 8, 128), (32, 32, 64), (16, 1, 128), (4, 2, 16)])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if head_dim == 16:
            dtype = "fp32"
        seqs = _between(rng, 1, 256)
        groups = rng.randint(1, max(1, min(6, seqs // 2)))
        private = rng.randint(0, max(0, seqs - 2 * groups) // 2)
        # CUDA-core paths and one-head-per-group layouts cost more per token
        most = 2048 if dtype == "fp32" or kv_heads == 32 else 30000
        prefix = _between(rng, 16, most)
        suffix = _between(rng, 1, 200 if most == 2048 else 1000)
        while seqs * (prefix + suffix) * heads * head_dim > 256 * 30000 * 32 * 128:
            prefix = max(16, prefix // 2)
        return {k: v for k, v in _attn("", dtype, heads, kv_heads, head_dim, seqs, groups,
                                       private, prefix, suffix).items() if k != "name"}
    vocab = _between(rng, 100, 200000)
    rows = _between(rng, 1, max(1, min(256, 256 * 128256 // vocab)))
    c = _samp("", rng.choice(["bf16", "fp16", "fp32"]), rows, vocab,
              round(rng.uniform(0.2, 1.6), 3), rng.choice([0, 0, _between(rng, 1, 1000)]),
              rng.choice([1.0, round(rng.uniform(0.05, 0.999), 3)]),
              rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.3), 4)]), rng.random() < 0.4)
    return {k: v for k, v in c.items() if k != "name"}


# ---------------------------------------------------------------- inputs
def _layout(case):
    """Who shares what, from the case's numbers alone: groups (lists of batch rows),
    their shared blocks and every row's length including the new token."""
    rng = random.Random(" ".join(str(case[k]) for k in
                                 ("heads", "head_dim", "seqs", "groups", "private", "prefix",
                                  "suffix")))
    n, g = case["seqs"], case["groups"]
    rows = list(range(n))
    rng.shuffle(rows)
    alone, rows = rows[:case["private"]], rows[case["private"]:]
    cuts = sorted(rng.sample(range(1, len(rows)), g - 1)) if g > 1 else []
    groups = [rows[a:b] for a, b in zip([0] + cuts, cuts + [len(rows)])]
    most = max(1, case["prefix"] // BLOCK)
    blocks = [most] + [max(1, int(most * rng.uniform(0.25, 1.0))) for _ in groups[1:]]
    lens = [0] * n
    for rs, p in zip(groups, blocks):
        for r in rs:
            lens[r] = p * BLOCK + rng.randint(1, case["suffix"])
    for r in alone:
        lens[r] = rng.randint(1, 2 * case["suffix"])
    return groups, blocks, lens


def _prepare_attention(case, seed):
    groups, blocks, lens = _layout(case)
    dev, dt = "cuda", DTYPES[case["dtype"]]
    H, Kh, D, n = case["heads"], case["kv_heads"], case["head_dim"], case["seqs"]
    row_blocks = [-(-x // BLOCK) for x in lens]
    shared = [0] * n
    for rs, p in zip(groups, blocks):
        for r in rs:
            shared[r] = p
    total = sum(blocks) + sum(a - b for a, b in zip(row_blocks, shared))
    ids = np.random.default_rng(seed).permutation(total + 8)  # scattered over the pool
    table = np.zeros((n, max(row_blocks)), dtype=np.int32)
    at = 0
    for rs, p in zip(groups, blocks):
        table[rs, :p] = ids[at:at + p]
        at += p
    for r in range(n):
        own_blocks = row_blocks[r] - shared[r]
        table[r, shared[r]:row_blocks[r]] = ids[at:at + own_blocks]
        at += own_blocks
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dt)

    st = {"case": case, "q": normal(n, H, D, scale=1.5), "k": normal(total + 8, BLOCK, Kh, D),
          "v": normal(total + 8, BLOCK, Kh, D), "table": torch.from_numpy(table).to(dev),
          "lens": torch.tensor(lens, dtype=torch.int32, device=dev), "scale": D ** -0.5}
    if own:
        from agentserve_b200 import ops
        # kept from step to step while the batch stays the same
        st["plan"] = ops.shared_prefix_plan(groups, blocks, row_blocks, H, Kh, D, dt, dev)
        st["ws"] = ops.new_shared_prefix_workspace(st["plan"])
    else:
        # the same knowledge as index tensors: members of every group (padded with row
        # 0), shared blocks of every group, and each row's place among them
        wide, deep = max(map(len, groups)), max(blocks)
        members = np.zeros((len(groups), wide), dtype=np.int64)
        first = np.zeros((len(groups), deep), dtype=np.int64)
        place = np.zeros((n, 2), dtype=np.int64)
        for i, (rs, p) in enumerate(zip(groups, blocks)):
            members[i, :len(rs)] = rs
            first[i, :p] = table[rs[0], :p]
            place[rs, 0], place[rs, 1] = i, np.arange(len(rs))
        st["members"], st["first"] = torch.from_numpy(members).to(dev), torch.from_numpy(first).to(dev)
        st["place"] = torch.from_numpy(place).to(dev)
        st["shared"] = torch.tensor(shared, device=dev) * BLOCK
        st["group_len"] = torch.tensor(blocks, device=dev) * BLOCK
        st["most_own"] = max((a - b) * BLOCK for a, b in zip(row_blocks, shared))
    return st


def _prepare_sample(case, seed):
    dev = "cuda"
    R, V = case["rows"], case["vocab"]
    g = torch.Generator(device=dev).manual_seed(seed)
    # a bulk of unlikely tokens and a few dozen likely ones, sharper in some rows
    x = torch.randn(R, V, generator=g, device=dev) * 2.2
    few = min(V, 64)
    likely = torch.randint(0, V, (R, few), generator=g, device=dev)
    sharp = 0.3 + torch.rand(R, 1, generator=g, device=dev)
    lift = 14.0 * torch.arange(1, few + 1, device=dev, dtype=torch.float32) ** -0.35
    x.scatter_add_(1, likely, sharp * lift)
    def rows(value, dtype):
        return torch.full((R,), value, dtype=dtype, device=dev)
    st = {"case": case, "logits": x.to(DTYPES[case["dtype"]]),
          "u": torch.rand(R, generator=g, device=dev),
          "temperature": rows(case["temperature"], torch.float32),
          "top_k": rows(case["top_k"], torch.int32), "top_p": rows(case["top_p"], torch.float32),
          "min_p": rows(case["min_p"], torch.float32),
          "logprobs": torch.empty(R, dtype=torch.float32, device=dev)}
    if case["mixed"]:  # every request has its own settings; some switch a filter off
        pick = torch.rand(5, R, generator=g, device=dev)
        st["temperature"] *= 0.4 + 1.2 * pick[0]
        st["temperature"][pick[1] < 0.15] = 0.0
        st["top_k"] = torch.where(pick[2] < 0.5, 0, st["top_k"] + (60 * pick[2]).int()).int()
        st["top_p"] = torch.where(pick[3] < 0.3, 1.0, 0.5 + 0.5 * pick[3])
        st["min_p"] = torch.where(pick[4] < 0.6, 0.0, 0.1 * pick[4])
    return st


def prepare(case, seed):
    return (_prepare_attention if case["op"] == "attention" else _prepare_sample)(case, seed)


# ---------------------------------------------------------------- one pass
def _plain_attention(st):
    c = st["case"]
    n, H, Kh, D = c["seqs"], c["heads"], c["kv_heads"], c["head_dim"]
    G = H // Kh
    q = (st["q"].float() * st["scale"]).view(n, Kh, G, D)
    # shared part, once per group: [groups, kv heads, members * G, keys]
    i, wide = st["members"].shape
    qs = q[st["members"]].permute(0, 2, 1, 3, 4).reshape(i, Kh, wide * G, D)
    k = st["k"][st["first"]].float().view(i, -1, Kh, D).permute(0, 2, 3, 1)
    v = st["v"][st["first"]].float().view(i, -1, Kh, D).permute(0, 2, 1, 3)
    s = qs @ k
    keys = torch.arange(s.shape[-1], device=s.device)
    s = s.masked_fill_(keys >= st["group_len"].view(-1, 1, 1, 1), float("-inf"))
    m1 = s.amax(-1, keepdim=True)
    s = (s - m1).exp_()
    l1, o1 = s.sum(-1, keepdim=True), s @ v

    def of_row(x):  # [groups, Kh, wide * G, *] -> [rows, Kh, G, *]
        x = x.view(i, Kh, wide, G, -1).transpose(1, 2)
        return x[st["place"][:, 0], st["place"][:, 1]]

    alone = (st["shared"] == 0).view(-1, 1, 1, 1)
    m1, l1, o1 = of_row(m1).masked_fill(alone, float("-inf")), of_row(l1), of_row(o1)
    # every row's own part
    at = torch.arange(st["most_own"], device=q.device) + st["shared"].view(-1, 1)
    last = st["table"].shape[1] - 1
    block = st["table"].gather(1, (at // BLOCK).clamp_(max=last)).long()
    k = st["k"][block, at % BLOCK].float().permute(0, 2, 3, 1)
    v = st["v"][block, at % BLOCK].float().permute(0, 2, 1, 3)
    s = q @ k
    s = s.masked_fill_((at >= st["lens"].view(-1, 1)).view(n, 1, 1, -1), float("-inf"))
    m2 = s.amax(-1, keepdim=True)
    s = (s - m2).exp_()
    l2, o2 = s.sum(-1, keepdim=True), s @ v
    # joined
    m = torch.maximum(m1, m2)
    w1, w2 = (m1 - m).exp(), (m2 - m).exp()
    o = (w1 * o1 + w2 * o2) / (w1 * l1 + w2 * l2)
    return o.reshape(n, H * D).to(st["q"].dtype)


def _plain_sample(st):
    # 64 bits: a token is chosen by comparing long sums that lie next to one another
    x = st["logits"].float().nan_to_num(0.0, 1e4, -1e4)
    greedy = st["temperature"] <= 1e-6
    t = st["temperature"].double().masked_fill(greedy, 1.0).view(-1, 1)
    val, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = ((val.double() - val[:, :1].double()) / t).exp_()
    rank = torch.arange(x.shape[1], device=x.device)
    k = st["top_k"].long()
    k = torch.where((k <= 0) | (k > x.shape[1]), x.shape[1], k).view(-1, 1)
    wk = w.masked_fill(rank >= k, 0.0)
    cum = wk.cumsum(1)
    p = st["top_p"].double().view(-1, 1)
    before = torch.cat([torch.zeros_like(cum[:, :1]), cum[:, :-1]], 1)
    keep = (before < p * cum[:, -1:]) | (p >= 1.0)
    keep &= w >= st["min_p"].double().view(-1, 1)
    keep |= rank == 0
    keep &= rank < k
    keep &= (rank == 0) | ~greedy.view(-1, 1)
    wi = torch.zeros_like(w).scatter_(1, order, w.masked_fill(~keep, 0.0))
    cum = wi.cumsum(1)
    total = cum[:, -1:]
    token = (cum <= st["u"].double().view(-1, 1) * total).sum(1)
    last = torch.where(wi > 0, rank, 0).amax(1)
    token = torch.minimum(token, last)
    st["logprobs"].copy_((wi.gather(1, token.view(-1, 1)) / total).log().view(-1))
    return token, st["logprobs"]


def run(state):
    if state["case"]["op"] == "attention":
        if own:
            from agentserve_b200 import ops
            return ops.shared_prefix_decode_attention(
                state["q"], state["k"], state["v"], state["table"], state["lens"],
                state["plan"], state["scale"], state["ws"])
        return _plain_attention(state)
    if own:
        from agentserve_b200 import ops
        return ops.sample_tokens(state["logits"], state["u"], state["temperature"],
                                 state["top_k"], state["top_p"], state["min_p"],
                                 logprobs=state["logprobs"]), state["logprobs"]
    return _plain_sample(state)


def work(case):
    es = DTYPES[case["dtype"]].itemsize
    if case["op"] == "attention":
        groups, blocks, lens = _layout(case)
        H, Kh, D = case["heads"], case["kv_heads"], case["head_dim"]
        tokens = sum(lens) - sum((len(rs) - 1) * p * BLOCK for rs, p in zip(groups, blocks))
        return {"bytes": es * (2 * tokens * Kh * D + 2 * case["seqs"] * H * D)
                + 4 * (-(-tokens // BLOCK) + case["seqs"]),
                "flops": 4 * H * D * sum(lens)}
    # every logit is read once; a scale, an exponential and a sum each
    R, V = case["rows"], case["vocab"]
    return {"bytes": R * V * es + R * (5 * 4 + 8 + 4), "flops": 3 * R * V}


# ---------------------------------------------------------------- the definition
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "attention":
        H, Kh, D = case["heads"], case["kv_heads"], case["head_dim"]
        out = torch.empty(case["seqs"], H, D, dtype=torch.float64, device="cuda")
        kf, vf = st["k"].view(-1, Kh, D), st["v"].view(-1, Kh, D)
        for b, n in enumerate(st["lens"].tolist()):  # one sequence after the other, whole
            pos = torch.arange(n, device="cuda")
            slot = st["table"][b].long()[pos // BLOCK] * BLOCK + pos % BLOCK
            for h in range(Kh):
                qh = st["q"][b, h * (H // Kh):(h + 1) * (H // Kh)].double()
                s = qh @ kf[slot, h].double().T * st["scale"]
                out[b, h * (H // Kh):(h + 1) * (H // Kh)] = torch.softmax(s, -1) @ vf[slot, h].double()
        return out.view(case["seqs"], H * D)
    x = st["logits"].float().cpu().numpy().astype(np.float64)
    x = np.nan_to_num(x, nan=0.0, posinf=1e4, neginf=-1e4)
    arg = {k: st[k].cpu().numpy().astype(np.float64) for k in
           ("u", "temperature", "top_k", "top_p", "min_p")}
    tokens, logs = [], []
    for r, row in enumerate(x):
        order = np.argsort(-row, kind="stable")
        if arg["temperature"][r] <= 1e-6:
            tokens.append(order[0])
            logs.append(0.0)
            continue
        w = np.exp((row[order] - row[order[0]]) / arg["temperature"][r])
        n = len(row)
        if 0 < arg["top_k"][r] < n:
            n = int(arg["top_k"][r])
        cum = np.cumsum(w[:n])
        kept = n
        if arg["top_p"][r] < 1.0:
            kept = min(kept, int(np.searchsorted(cum, arg["top_p"][r] * cum[-1], side="left")) + 1)
        kept = max(1, min(kept, int(np.count_nonzero(w[:n] >= arg["min_p"][r]))))
        by_index = np.sort(order[:kept])
        wi = np.exp((row[by_index] - row[order[0]]) / arg["temperature"][r])
        cum = np.cumsum(wi)
        at = min(int(np.searchsorted(cum, arg["u"][r] * cum[-1], side="right")),
                 int(np.flatnonzero(wi > 0)[-1]))
        tokens.append(by_index[at])
        logs.append(np.log(wi[at] / cum[-1]))
    return (torch.tensor(np.array(tokens, dtype=np.int64)),
            torch.tensor(np.array(logs, dtype=np.float64)))
