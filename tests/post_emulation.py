"""PyTorch stand-ins of the post-training and 8-bit activation kernels for CPU tests of the fused engine's host code
(``fused_emulation`` has those of the other kernels)."""
from __future__ import annotations

import torch

import fused_emulation
import post_oracle as O


def token_logprobs(logits, V, targets, ignore_index=-100, grad=None):
    logp, lse, g = O.logprobs(logits, V, targets, ignore_index)
    if grad is not None:
        g = g.to(grad.dtype)
        grad.zero_()
        grad[:, :V].copy_(g)
    return logp.float(), lse.float()


def policy_loss(logits, V, targets, old_logp, advantages, ref_logp=None, weights=None, clip_low=0.2, clip_high=0.2,
                kl_coef=0.0, grad_scale=None, ignore_index=-100, grad=None):
    logp, _, g = O.logprobs(logits, V, targets, ignore_index)
    loss, stats, d = O.policy(logp, targets != ignore_index, old_logp, advantages, ref_logp, weights, clip_low, clip_high,
                              kl_coef)
    d = d * (1.0 if grad_scale is None else grad_scale.double())
    out = torch.empty_like(logits) if grad is None else grad
    out.zero_()
    out[:, :V].copy_((d[:, None] * g).to(out.dtype))
    return loss.float(), stats.float(), logp.float(), out


def preference_loss(logp, targets, ref_logp=None, beta=0.1, label_smoothing=0.0, ignore_index=-100):
    return tuple(t.float() for t in O.preference(logp, targets, ref_logp, beta, label_smoothing, ignore_index))


def act8_pack(x):
    codes, es, bad = O.act8_codes(x)
    return codes.to(torch.int8), torch.where(bad, torch.full_like(es, 255), es + 127).to(torch.uint8)


def act8_unpack(q, e, dtype=torch.bfloat16):
    bad = e == 255
    return O.act8_values(q.long(), torch.where(bad, 127, e.long()) - 127, bad, dtype).to(dtype)


def act8_unpack_gelu(q, e, dtype=torch.bfloat16):
    x = act8_unpack(q, e, torch.float32)
    return O.gelu(x).to(dtype), x.to(dtype)


def layernorm_fwd_act8(x, w, b, eps=1e-5, dtype=torch.bfloat16):
    mean = x.mean(-1, keepdim=True)
    rstd = torch.rsqrt(x.var(-1, unbiased=False, keepdim=True) + eps)
    xh = (x - mean) * rstd
    return ((xh * w + b).to(dtype), *act8_pack(xh), rstd[:, 0])


def layernorm_bwd_act8(dy, q, e, rstd, w, b, dres_in, dres, dres16, dgamma, dbeta):
    xh = act8_unpack(q, e, torch.float32)
    dgamma.add_((dy * xh).sum(0))
    dbeta.add_(dy.sum(0))
    gw = dy * w
    new = dres_in + rstd[:, None] * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    dres.copy_(new)
    dres16.copy_(new.to(dres16.dtype))
    return (xh * w + b).to(dres16.dtype)


NAMES = ["token_logprobs", "policy_loss", "preference_loss", "act8_pack", "act8_unpack", "act8_unpack_gelu",
         "layernorm_fwd_act8", "layernorm_bwd_act8"]


def emulate(monkeypatch) -> None:
    """``fused_emulation.emulate`` and the stand-ins above."""
    from heiretsu_b200.models import objectives
    from heiretsu_b200.ops import kernels as K

    fused_emulation.emulate(monkeypatch)
    for name in NAMES:
        monkeypatch.setattr(K, name, globals()[name])
    monkeypatch.setattr(objectives, "_fused", lambda model, idx: model.fused)
