"""What the tests of the 8-bit attention backward share: a block whose scores are as sharp as a trained model's, and its
gradient by the formula on the Q/K/V that the backward reads."""
from __future__ import annotations

import math

import torch

import post_oracle as O

STD = 2.0  # of the Q and K channels: scores of standard deviation 4


def block(offset: float, device="cpu", dtype16=torch.bfloat16, nh=4, dropout=0.0):
    """(block of head_dim 64, its input [B T, H], B, T): Q and K channels of standard deviation ``STD``, the fourth K
    channel of every head offset by ``offset``, as trained models have."""
    from heiretsu_b200.config import GPTConfig
    from heiretsu_b200.models.gpt import GPT
    from heiretsu_b200.parallel.flat import FlatParams

    B, T, H = 2, 192, 64 * nh
    torch.manual_seed(3)
    m = GPT(GPTConfig(block_size=T, vocab_size=64, n_layer=1, n_head=nh, n_embed=H, dropout=dropout)).to(device)
    blk = m.tr.h[0]
    with torch.no_grad():
        w, b = blk.attn.c_attn.weight, blk.attn.c_attn.bias
        w.normal_(0, 1 / math.sqrt(H))
        w[:2 * H].mul_(STD)
        b[H:2 * H].view(nh, 64)[:, 3] = offset
    blk._flat = FlatParams(m, torch.device(device), dtype16=dtype16)
    return blk, torch.randn(B * T, H, device=device), B, T


@torch.no_grad()
def error(monkeypatch, offset, device="cpu", dtype16=torch.bfloat16, drop=None):
    """(relative error of the attention's gradient against the formula on the Q/K/V it was given, and its bound)."""
    from heiretsu_b200.models import fused as FZ
    from heiretsu_b200.ops import dropout_ref as DR
    from heiretsu_b200.ops import kernels as K

    blk, x, B, T = block(offset, device, dtype16, dropout=drop or 0.0)
    nh, H = blk.attn.nh_tp, x.shape[1]
    mask = None
    if drop:
        seed = torch.tensor([41], dtype=torch.int32, device=device)
        blk._hb_drop_now = (seed, 0, drop)
        mask = DR.attention_mask(41, 0, B, nh, T, drop, 0, nh).to(device)
    seen = []
    real = K.attention_bwd
    monkeypatch.setattr(K, "attention_bwd", lambda *a, **k: seen.append((a[0].clone(), a[2].clone(), real(*a, **k)))
                        or seen[-1][2])
    _, saved = FZ._attn_fwd(blk, x, B, T, True, act8=True)
    dres = torch.randn(B * T, H, device=device)
    FZ._attn_bwd(blk, saved, dres, dres.to(dtype16), B, T, {})
    (qkv, dout, got), = seen
    want = O.attention_grad(qkv, dout, B, T, nh, 64, mask)
    # y, P and dS (or their 32-bit stand-ins) are rounded to 16 bits: errors of half a step each, which an offset of one of
    # a head's 64 K channels multiplies there by offset / STD
    bound = 3 * O.EPS[dtype16] * (1 + offset / STD / 8)
    return ((got.double() - want).norm() / want.norm()).item(), bound
