"""Tokens of the fused mixture of experts whose router logits are no numbers."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _block(E, K, H=128):
    from heiretsu_b200.config import GPTConfig
    from heiretsu_b200.models.gpt import BlockMoE
    from heiretsu_b200.parallel.flat import FlatParams

    torch.manual_seed(0)
    blk = BlockMoE(GPTConfig(block_size=256, vocab_size=100, n_layer=2, n_head=2, n_embed=H, num_experts=E, top_k=K)).cuda()
    with torch.no_grad():
        blk.moe.router.gate.weight.mul_(5.0)
    FlatParams(blk, torch.device("cuda"))
    return blk


@pytest.mark.parametrize("E,K,N", [(8, 2, 300), (4, 1, 5), (4, 4, 1), (64, 8, 130)])
def test_a_broken_token_leaves_the_others_alone(E, K, N):
    """NaN and infinities in some tokens' rows: these come out as NaN, every other row as it would without them, and every
    choice has an expert and a place of its own."""
    from heiretsu_b200.models.fused_moe import moe_sublayer_fwd
    from heiretsu_b200.ops._C import check_status

    blk = _block(E, K)
    x = torch.randn(N, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(N))
    want, _, _ = moe_sublayer_fwd(blk, None, x, keep=False)
    bad = torch.zeros(N, dtype=torch.bool, device="cuda")
    for i, value in ((0, math.nan), (N // 2, math.inf), (N - 1, -math.inf)):
        x[i, 7] = value
        bad[i] = True
    out, _, saved = moe_sublayer_fwd(blk, None, x, keep=True)
    check_status()
    assert bool(out[bad].isnan().any(1).all())
    assert torch.equal(out[~bad], want[~bad])
    probs, topi, topw, counts, off, _, pos = saved[4][:7]
    topi, pos = topi.view(N, K).long(), pos.long()
    assert bool(((topi >= 0) & (topi < E)).all()) and torch.equal(topi[bad], torch.arange(K, device="cuda").expand(int(bad.sum()), K))
    assert counts.tolist() == torch.bincount(topi.view(-1), minlength=E).tolist()
    e = topi.view(-1)
    assert bool(((pos >= off[e]) & (pos < off[e] + counts[e])).all()) and pos.unique().numel() == N * K
