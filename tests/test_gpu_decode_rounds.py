"""Decode attention over splits that end inside a round of the warps that read them (four
blocks a round): many blocks on every SM and many calls, all of the same bits and right."""

import pytest
import torch

from agentserve_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("H,Kh,D,dtype", [(32, 8, 64, torch.bfloat16), (32, 8, 128, torch.float16),
                                          (6, 3, 128, torch.bfloat16)])
@pytest.mark.parametrize("bps", [0, 5, 11, 13])
def test_rounds_with_warps_without_a_block(H, Kh, D, dtype, bps):
    B, NB = 64, 900
    g = torch.Generator(device=DEV).manual_seed(D + bps)
    lens = torch.tensor([1 + (37 * i) % 1000 for i in range(B)], dtype=torch.int32, device=DEV)
    table = torch.randint(0, NB, (B, 63), generator=g, device=DEV, dtype=torch.int32)
    q = (8 * torch.randn(B, H, D, generator=g, device=DEV)).to(dtype)
    k, v = (torch.randn(NB, 16, Kh, D, generator=g, device=DEV).to(dtype) for _ in range(2))
    ws = ops.new_decode_workspace(B, H, Kh, D, 63, bps, DEV)

    def run():
        return ops.paged_decode_attention(q, k, v, table, lens, D ** -0.5, bps, ws)
    first = run()
    # probabilities and result rounded to the type, half a step each; fp32 sums of up to 1000
    # keys and D products, and 2^-24 where fp16 has no smaller step
    half = torch.finfo(dtype).eps / 2
    for b in range(B):
        n = int(lens[b])
        at = torch.arange(n, device=DEV)
        slot = table[b].long()[at // 16] * 16 + at % 16
        kb, vb = (x.view(-1, Kh, D)[slot].double().repeat_interleave(H // Kh, 1) for x in (k, v))
        s = torch.einsum("hd,nhd->hn", q[b].double(), kb) * D ** -0.5
        p = torch.softmax(s, -1)
        ref, A = (torch.einsum("hn,nhd->hd", p, x) for x in (vb, vb.abs()))
        S = float(torch.einsum("hd,nhd->hn", q[b].double().abs(), kb.abs()).max() * D ** -0.5)
        tol = (2 * (n + D * S + 64) * 2.0 ** -24 + half) * A + half * ref.abs() + 2.0 ** -24
        assert ((first[b].view(H, D).double() - ref).abs() <= tol).all(), b
    for _ in range(100):
        assert torch.equal(run(), first)
    assert ops.device_status(clear=True) == 0
