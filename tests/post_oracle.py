"""64-bit oracles of the post-training losses and of the 8-bit activation format, and the error bounds that the
GPU tests hold the kernels to. Everything here runs on any device."""
from __future__ import annotations

import torch

IGNORE = -100
EPS = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}  # half a step, relative
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}  # half the least step


def logprobs(logits, V, targets, ignore=IGNORE):
    """(logp, lse, unit gradient [M, V]) in 64 bits; zeros in ignored rows."""
    x = logits[:, :V].double()
    live = targets != ignore
    top = x.amax(1, keepdim=True)
    y = x - top  # first: next to a mask of the type's lowest value, log of the sum would vanish even in 64 bits
    rest = torch.logsumexp(y, 1)
    lse = top[:, 0] + rest
    at = torch.arange(x.shape[0], device=x.device), targets.clamp(0, V - 1)
    logp = y[at] - rest
    g = -torch.exp(y - rest[:, None])
    g[at] += 1
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    return torch.where(live, logp, zero), torch.where(live, lse, zero), torch.where(live[:, None], g, zero)


def policy(logp, live, old, adv, ref=None, weights=None, lo=0.2, hi=0.2, kl_coef=0.0):
    """(loss, stats [2], dloss/dlogp) in 64 bits, through autograd on the formula."""
    lp = logp.detach().double().requires_grad_(True)
    w = live.double() / live.sum().clamp_min(1) if weights is None else weights.double() * live
    n = adv.numel()
    A = adv.double().repeat_interleave(lp.numel() // n) if n else adv.double()
    with torch.enable_grad():
        r = torch.exp(torch.where(live, lp - old.double(), torch.zeros_like(lp)))
        free, kept = r * A, r.clamp(1 - lo, 1 + hi) * A
        clipped = kept < free
        per = -torch.where(clipped, kept.detach(), free)
        kl = torch.zeros_like(lp)
        if ref is not None:
            u = torch.where(live, ref.double() - lp, torch.zeros_like(lp))
            kl = torch.expm1(u) - u
            per = per + kl_coef * kl
        loss = (w * per).sum()
        (d,) = torch.autograd.grad(loss, lp) if lp.numel() else (lp.detach(),)
    return loss.detach(), torch.stack([(w * kl).sum(), (w * clipped).sum()]).detach(), d


def preference(logp, targets, ref=None, beta=0.1, smoothing=0.0, ignore=IGNORE):
    """(loss, rewards [2, P], dlogp) in 64 bits, through autograd on the formula."""
    lp = logp.detach().double().requires_grad_(True)
    P = lp.shape[0] // 2
    live = targets != ignore
    with torch.enable_grad():
        d = lp if ref is None else lp - ref.double()
        R = beta * torch.where(live, d, torch.zeros_like(d)).sum(1).view(2, P)
        z = R[0] - R[1]
        ls = torch.nn.functional.logsigmoid
        loss = (-(1 - smoothing) * ls(z) - smoothing * ls(-z)).mean()
        (g,) = torch.autograd.grad(loss, lp)
    return loss.detach(), R.detach(), g


def lse_bound(lse, V):
    """How far a 32-bit log-sum-exp over V terms may be: each exponential is off by at most 2 + 1.173 |arg| units in
    the last place (CUDA's bound for __expf), |arg| averaging at most log V under the softmax; a sum split over at
    least 128 threads adds at most V / 128 + 16 roundings; lse itself is rounded, as is max + log."""
    terms = (2 + 1.173 * torch.log(torch.tensor(float(V))).item()) * 2.0 ** -23
    return terms + (V / 128 + 16) * 2.0 ** -24 + 4 * 2.0 ** -24 * lse.abs()


def grad_bound(g, coef, logits, lse, V, dtype):
    """Element-wise bound of coef (onehot - p): the output's rounding, p's relative error (the exponential's, and lse's
    as an exponent), and four roundings of the products."""
    arg = (logits.double()[:, :V] - lse[:, None]).abs()
    arg = torch.where(torch.isfinite(arg), arg, torch.zeros_like(arg))
    rel = (2 + 1.173 * arg) * 2.0 ** -23 + lse_bound(lse, V)[:, None]
    p = torch.exp(logits.double()[:, :V] - lse[:, None])
    return EPS[dtype] * g.abs() + TINY[dtype] + coef.abs()[:, None] * (p * rel + 4 * 2.0 ** -24)


# ---- 8-bit activations -----------------------------------------------------------
def act8_codes(x):
    """(codes int64 [M, N], e [M, blocks], NaN blocks [M, blocks]) of the format, in 64 bits."""
    M, N = x.shape
    xd = x.double()
    codes = torch.zeros(M, N, dtype=torch.int64, device=x.device)
    nb = (N + 127) // 128
    es = torch.zeros(M, nb, dtype=torch.int64, device=x.device)
    bad = torch.zeros(M, nb, dtype=torch.bool, device=x.device)
    for k in range(nb):
        xb = xd[:, 128 * k:128 * k + 128]
        bad[:, k] = ~torch.isfinite(xb).all(1)
        xb = torch.where(bad[:, k:k + 1], torch.zeros_like(xb), xb)
        top = xb.abs().amax(1)
        e = torch.full((M,), -126, dtype=torch.int64, device=x.device)
        for cand in range(-126, 123):  # the least exponent that holds the largest value
            e = torch.where(top > 127 * 2.0 ** (cand), torch.full_like(e, cand + 1), e)
        es[:, k] = e
        codes[:, 128 * k:128 * k + 128] = torch.round(xb * torch.exp2(-e.double())[:, None]).long()
    return codes, es, bad


def act8_values(codes, es, bad, dtype=torch.float64):
    """The values the codes stand for, clamped to dtype's finite range; NaN in bad blocks."""
    block = torch.arange(codes.shape[1], device=codes.device) // 128
    v = codes.double() * torch.exp2(es.double())[:, block]
    if dtype != torch.float64:
        v = v.clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max)
    return torch.where(bad[:, block], torch.full_like(v, float("nan")), v)


def gelu(x):
    """0.5 x (1 + tanh u) as x sigmoid(2u): the sum 1 + tanh u keeps no digit in 64 bits below u = -18."""
    x = x.double()
    return x * torch.sigmoid(2 * 0.7978845608028654 * (x + 0.044715 * x ** 3))


def attention_grad(qkv, dout, B, T, nh, dh, mask=None):
    """Gradient [B T, 3 nh dh] of causal softmax attention in 64 bits, by the formula: with P the softmax and y = (m P) V,
    dP = m dy V^T, dS = P (dP - sum P dP). ``mask`` [B, nh, T, T]: the dropout factors m."""
    q, k, v = qkv.double().view(B, T, 3, nh, dh).permute(2, 0, 3, 1, 4).unbind(0)
    do = dout.double().view(B, T, nh, dh).transpose(1, 2)
    s = q @ k.transpose(-1, -2) / dh ** 0.5
    s = s.masked_fill(torch.ones(T, T, dtype=torch.bool, device=s.device).triu(1), float("-inf"))
    p = torch.softmax(s, -1)
    m = torch.ones_like(p) if mask is None else mask.double()
    dp = m * (do @ v.transpose(-1, -2))
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / dh ** 0.5
    d = torch.stack([ds @ k, ds.transpose(-1, -2) @ q, (m * p).transpose(-1, -2) @ do])
    return d.permute(1, 3, 0, 2, 4).reshape(B * T, 3 * nh * dh)
