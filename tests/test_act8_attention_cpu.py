"""Attention backward from 8-bit Q/K/V: consistent with the scores it reads. The stand-ins here follow the kernels' contract,
with the statistics handed over (those of fused_emulation evaluate the softmax again and cannot show a mismatch)."""
import math

import pytest
import torch

import act8_attention as A
import post_emulation
from heiretsu_b200.ops import dropout_ref as DR

LOG2E = math.log2(math.e)


def scores(qkv, B, T, nh, dh):
    q, k, v = qkv.float().view(B, T, 3, nh, dh).permute(2, 0, 3, 1, 4).unbind(0)
    s = q @ k.transpose(-1, -2) * (LOG2E / dh ** 0.5)
    return q, k, v, s.masked_fill(torch.ones(T, T, dtype=torch.bool).triu(1), float("-inf"))


def keep(drop, B, nh, T):
    if drop is None:
        return torch.ones(())
    seed, site, p, h0, nht = drop
    return DR.attention_mask(int(seed.reshape(-1)[0]), site, B, nh, T, p, h0, nht).float()


def attention_fwd(qkv, B, T, nh, out=None, drop=None, head_dim=64):
    _, _, v, s = scores(qkv, B, T, nh, head_dim)
    lse2 = torch.logsumexp(s / LOG2E, -1) * LOG2E
    y = (keep(drop, B, nh, T) * torch.exp2(s - lse2[..., None])) @ v
    nlse = torch.zeros(B, nh, (T + 127) // 128 * 128)
    nlse[..., :T] = -lse2
    y = y.transpose(1, 2).reshape(B * T, nh * head_dim).to(qkv.dtype)
    return (y if out is None else out.copy_(y)), nlse


def attention_bwd(qkv, out, dout, lse, B, T, nh, dqkv=None, drop=None, head_dim=64):
    q, k, v, s = scores(qkv, B, T, nh, head_dim)
    do, y = (t.float().view(B, T, nh, head_dim).transpose(1, 2) for t in (dout, out))
    p, m = torch.exp2(s + lse[..., :T, None]), keep(drop, B, nh, T)
    ds = p * (m * (do @ v.transpose(-1, -2)) - (do * y).sum(-1, keepdim=True)) / head_dim ** 0.5
    d = torch.stack([ds @ k, ds.transpose(-1, -2) @ q, (m * p).transpose(-1, -2) @ do])
    return d.permute(1, 3, 0, 2, 4).reshape(B * T, 3 * nh * head_dim).to(qkv.dtype)


@pytest.mark.parametrize("drop", [None, 0.2])
@pytest.mark.parametrize("offset", [0.0, 20.0, 40.0])
def test_backward_of_the_restored_scores(monkeypatch, offset, drop):
    from heiretsu_b200.ops import kernels as K

    post_emulation.emulate(monkeypatch)
    monkeypatch.setattr(K, "attention_fwd", attention_fwd)
    monkeypatch.setattr(K, "attention_bwd", attention_bwd)
    err, bound = A.error(monkeypatch, offset, drop=drop)
    assert err <= bound, (err, bound)
