"""PyTorch stand-ins of the decoding kernels for CPU tests of the decoder's host code (``fused_emulation`` has those of
the other kernels)."""
from __future__ import annotations

import torch

import decode_oracle as O
import fused_emulation


def kv_write(k, v, slots, k_pages, v_pages, k_exp=None, v_exp=None):
    live = slots >= 0
    assert slots[live].unique().numel() == int(live.sum()), "two tokens in one slot"
    assert bool((slots < k_pages.shape[0] * k_pages.shape[2]).all())
    c = O.Cache.__new__(O.Cache)
    c.bits, c.size = 8 if k_exp is not None else 16, k_pages.shape[2]
    c.pools = dict(k_pages=k_pages, v_pages=v_pages, k_exp=k_exp, v_exp=v_exp)
    c.put(slots[live], k[live], v[live])


def kv_read(slots, k_pages, v_pages, k_exp=None, v_exp=None, dtype=None):
    page, at = slots.clamp_min(0) // k_pages.shape[2], slots.clamp_min(0) % k_pages.shape[2]
    out = []
    for pool, exp in ((k_pages, k_exp), (v_pages, v_exp)):
        x = pool[page, :, at]
        if exp is not None:
            x = (x.double() * torch.exp2(exp[page, :, at].double() - 127)[..., None]).to(dtype or torch.bfloat16)
        out.append(x * (slots >= 0)[:, None, None].to(x.dtype))
    return tuple(out)


def decode_attention(q, k_pages, v_pages, table, lengths, k_exp=None, v_exp=None, scale=None):
    size = k_pages.shape[2]
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2])
    for b, n in enumerate(lengths.tolist()):
        at = torch.arange(n)
        k, v = kv_read(table[b].long()[at // size] * size + at % size, k_pages, v_pages, k_exp, v_exp, torch.float32)
        o, e, _, _ = O.attention(q[b], k.double(), v.double(), q.shape[2] ** -0.5 if scale is None else scale)
        out[b], lse[b] = o.to(q.dtype), e.float()
    return out, lse


def sample_tokens(logits, V, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    return torch.tensor([O.sample_row(x[:V], float(r), temperature, top_k, top_p, min_p) for x, r in zip(logits, u)])


def attention_fwd(qkv, B, T, nh, out=None, drop=None, head_dim=64):
    """Rounded to qkv's type, whichever it is."""
    q, k, v = fused_emulation._qkv(qkv, B, T, nh, head_dim)
    y = fused_emulation._attn(q, k, v, T, drop, B, nh).transpose(1, 2).reshape(B * T, nh * head_dim)
    return y.to(qkv.dtype), None


def emulate(monkeypatch) -> None:
    from heiretsu_b200.ops import kernels as K

    fused_emulation.emulate(monkeypatch)
    for name in ("kv_write", "kv_read", "decode_attention", "sample_tokens", "attention_fwd"):
        monkeypatch.setattr(K, name, globals()[name])
