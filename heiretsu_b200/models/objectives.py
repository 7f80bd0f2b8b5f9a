"""Post-training objectives of the GPT model: token log-probabilities, a clipped policy loss with a KL
term, and a preference loss on pairs (the reference trains on next-token cross-entropy only).

``GPT.token_logprobs``, ``GPT.policy_loss`` and ``GPT.preference_loss`` call these. On the fused engine the head
(ln_f, lm_head GEMM, loss) is one autograd node over the kernels of csrc/post_loss.cu:

* log-probabilities with a gradient: one pass over the 16-bit logits writes logp and, in place, the unit gradient
  G = onehot - softmax. Whatever loss the caller builds, its gradient in the logits is diag(dlogp) G, and the factor
  goes to the small operands: d(hidden) = diag(dlogp) (G W) and dW = G^T (diag(dlogp) hidden), so the logits are not
  read a third time. In fp16, whose range does not hold G (a probability below 2^-25 is 0) nor dlogp times the hidden
  states under a loss scale, the gradient is formed in backward, dlogp and with it the loss scale included. Scoring
  without a gradient (a reference model, sampled tokens) only reads the logits;
* the policy loss is a function of each token alone, so one pass writes the loss terms and the complete gradient;
* the preference loss sums log-probabilities over sequences first and runs on them.

Elsewhere (CPU, fp32, tensor parallelism) the same formulas run in PyTorch on the plain modules. Fused tensor
parallelism shards the tokens of a batch over ranks and is refused here: use ``--engine plain``.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn.functional as F

from ..ops import gemm as G
from ..ops import kernels as K

IGNORE = -100


def _fused(model, idx: torch.Tensor) -> bool:
    if not (model.fused and idx.is_cuda):
        return False
    if getattr(getattr(model, "topo", None), "tp", 1) > 1:
        raise ValueError("post-training objectives on the fused engine need tp 1 (the plain engine runs them with tensor "
                         "parallelism)")
    return True


def _trunk(model, idx: torch.Tensor, fused: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """The residual stream behind the last block [B, T, H] and the summed MoE aux loss."""
    B, T = idx.shape
    if T > model.cfg.block_size:
        raise ValueError(f"input of {T} positions exceeds the model's block_size of {model.cfg.block_size}")
    if fused:
        from .fused import blocks_fused, embed_fused
        x = embed_fused(model.tr.wte.weight, model.tr.wpe.weight, idx)
        return blocks_fused(model.tr.h, x, model.cfg, recompute=getattr(model, "recompute", False),
                            act_bits=getattr(model, "act_bits", 16))
    from .gpt import run_blocks
    x = model.tr.wte(idx) + model.tr.wpe(torch.arange(T, device=idx.device))[None]
    return run_blocks(model.tr.h, x, model.recompute)


def _check(idx: torch.Tensor, targets: torch.Tensor, **per_token) -> None:
    if idx.dim() != 2 or targets.shape != idx.shape:
        raise ValueError(f"idx and targets must both be [B, T], got {tuple(idx.shape)} and {tuple(targets.shape)}")
    for name, t in per_token.items():
        if t is not None and t.shape != idx.shape:
            raise ValueError(f"{name} must be [B, T] like idx, got {tuple(t.shape)}")


def _check_policy(clip_low: float, clip_high: float, kl_coef: float) -> None:
    if not (0 <= clip_low <= 1 and 0 <= clip_high < math.inf):
        raise ValueError(f"clip_low must be in [0, 1] and clip_high finite and not negative, got {clip_low}, {clip_high}")
    if not math.isfinite(kl_coef):
        raise ValueError(f"kl_coef must be finite, got {kl_coef}")


def _check_preference(beta: float, label_smoothing: float) -> None:
    if not math.isfinite(beta):
        raise ValueError(f"beta must be finite, got {beta}")
    if not 0 <= label_smoothing <= 1:
        raise ValueError(f"label_smoothing must be in [0, 1], got {label_smoothing}")


def _flat32(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if t is None else t.reshape(-1).float().contiguous()


# ---- fused heads -----------------------------------------------------------------
def _logits(x, ln_w, ln_b, wte, V: int):
    from .fused import LN_EPS, _vpad
    dt = wte.w16.dtype
    xn, mean, rstd = K.layernorm_fwd(x, ln_w, ln_b, LN_EPS, dtype=dt)
    logits = torch.empty(x.shape[0], _vpad(V), device=x.device, dtype=dt)
    G.gemm(xn, wte.w16, logits, _vpad(V), G.EPI_BF16, False, False)
    return xn, mean, rstd, logits


def _head_grads(dl, V: int, xn, x, mean, rstd, ln_w, ln_b, wte, rows: Optional[torch.Tensor] = None) -> torch.Tensor:
    """d(x) from the logits' gradient ``diag(rows) dl`` (rows None: ones); parameter gradients go to ``main_grad``."""
    dxn = G.linear_dgrad(dl[:, :V], wte.w16, f32=True)
    if rows is not None:
        # the factors go to the operands that have H columns, not V. The scaled hidden states are rounded to
        # 16 bits once more (half a unit in the last place of the weight gradient's operand).
        dxn.mul_(rows[:, None])
        xn = torch.mul(xn, rows[:, None], out=torch.empty_like(xn))
    G.linear_wgrad(dl, xn, out=wte.main_grad, accumulate=True, n_rows=V)
    dx = torch.empty_like(x)
    dx16 = torch.empty(x.shape, device=x.device, dtype=xn.dtype)
    K.layernorm_bwd(dxn, x, mean, rstd, ln_w, torch.zeros_like(x), dx, dx16, ln_w.main_grad, ln_b.main_grad)
    return dx


class _HeadLogp(torch.autograd.Function):
    """ln_f -> lm_head -> log-probability of each row's target [M]."""

    @staticmethod
    def forward(ctx, x, ln_w, ln_b, wte, targets, V, with_grad):
        xn, mean, rstd, logits = _logits(x, ln_w, ln_b, wte, V)
        ctx.unit = logits.dtype != torch.float16
        logp, _ = K.token_logprobs(logits, V, targets, grad=logits if with_grad and ctx.unit else None)
        if with_grad:
            ctx.save_for_backward(x, xn, mean, rstd, logits, targets, logp)
            ctx.params, ctx.V = (ln_w, ln_b, wte), V
        return logp

    @staticmethod
    def backward(ctx, dlogp):
        x, xn, mean, rstd, dl, targets, logp = ctx.saved_tensors
        # an ignored row's log-probability is the constant 0, whatever comes for it: the derivative of sqrt(-logp) or
        # log(-logp) is infinite there, and 0 times infinity would reach every parameter
        rows = torch.where(targets != IGNORE, dlogp.float(), 0.0)
        if not ctx.unit:
            # the policy loss of the model against itself has ratios of exactly 1: its gradient at advantage 1 and
            # weight -dlogp is that of sum dlogp logp
            K.policy_loss(dl, ctx.V, targets, logp, torch.ones(1, device=dl.device), weights=-rows, grad=dl)
            rows = None
        dx = _head_grads(dl, ctx.V, xn, x, mean, rstd, *ctx.params, rows=rows)
        return dx, None, None, None, None, None, None


class _HeadPolicy(torch.autograd.Function):
    """ln_f -> lm_head -> policy loss; the gradient is written in the same pass, for the upstream gradient the caller
    is expected to send, and corrected in backward where that differs (as the cross-entropy head does)."""

    @staticmethod
    def forward(ctx, x, ln_w, ln_b, wte, targets, V, with_grad, old, adv, ref, weights, lo, hi, kl, hint, scale):
        xn, mean, rstd, logits = _logits(x, ln_w, ln_b, wte, V)
        expected = torch.full((1,), float(hint), device=x.device, dtype=torch.float32)
        if scale is not None:
            expected = expected * scale
        loss, stats, logp, grad = K.policy_loss(logits, V, targets, old, adv, ref_logp=ref, weights=weights,
                                                clip_low=lo, clip_high=hi, kl_coef=kl, grad_scale=expected,
                                                grad=logits)
        ctx.mark_non_differentiable(stats, logp)
        if with_grad:
            ctx.save_for_backward(x, xn, mean, rstd, grad, expected)
            ctx.params, ctx.V = (ln_w, ln_b, wte), V
        return loss, stats, logp

    @staticmethod
    def backward(ctx, dloss, _dstats, _dlogp):
        x, xn, mean, rstd, grad, expected = ctx.saved_tensors
        dl = K.cross_entropy_rescale_(grad, dloss.reshape(1).float().contiguous(), expected)
        dx = _head_grads(dl, ctx.V, xn, x, mean, rstd, *ctx.params)
        return (dx,) + (None,) * 15


class _Preference(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logp, targets, ref, beta, smoothing):
        loss, rewards, dlogp = K.preference_loss(logp, targets, ref_logp=ref, beta=beta, label_smoothing=smoothing)
        ctx.save_for_backward(dlogp)
        ctx.mark_non_differentiable(rewards)
        return loss, rewards

    @staticmethod
    def backward(ctx, dloss, _drewards):
        (dlogp,) = ctx.saved_tensors
        return dlogp * dloss, None, None, None, None


def _head_args(model, x: torch.Tensor, targets: torch.Tensor):
    x2 = x.reshape(-1, x.shape[-1])
    x2 = (x2 if x2.dtype == torch.float32 else x2.float()).contiguous()
    with_grad = torch.is_grad_enabled() and x2.requires_grad
    return (x2, model.tr.ln_f.weight, model.tr.ln_f.bias, model.lm_head.weight, targets.reshape(-1).contiguous(),
            model.cfg.vocab_size, with_grad)


# ---- formulas in PyTorch -------------------------------------------------------------
def _logp_plain(model, x: torch.Tensor, targets: torch.Tensor) -> torch.Tensor:
    logits = model.lm_head(model.tr.ln_f(x))
    V = logits.shape[-1]
    counts, known = targets != IGNORE, (targets >= 0) & (targets < V)
    logp = F.log_softmax(logits.float(), dim=-1).gather(-1, targets.clamp(0, V - 1)[..., None])[..., 0]
    # a target that is no token gives NaN, and so does its gradient: as with the kernels, the step is skipped
    return torch.where(counts, logp * torch.where(counts & ~known, float("nan"), 1.0), torch.zeros_like(logp))


def policy_loss_plain(logp, targets, old_logp, advantages, ref_logp, weights, clip_low, clip_high, kl_coef):
    """(loss, stats) of ``ops.kernels.policy_loss`` from log-probabilities [B, T], by autograd in them alone."""
    old_logp, advantages, ref_logp, weights = (None if t is None else t.detach()
                                               for t in (old_logp, advantages, ref_logp, weights))
    counts = targets != IGNORE
    zero = torch.zeros_like(logp)
    w = counts / counts.sum().clamp_min(1) if weights is None else torch.where(counts, weights.float(), zero)
    adv = advantages.float() if advantages.shape == logp.shape else advantages.float()[:, None].expand_as(logp)
    # a ratio past 32 bits (log-ratios from 89) stands for a finite number, which the clip range, an advantage or a weight
    # of 0 takes out, as in the kernel; infinity would leave NaN, here or in the exponential's derivative
    finite = lambda d, out: torch.where(counts, torch.where(out, d.clamp(max=80), d), zero)  # noqa: E731
    ratio = torch.exp(finite(logp - old_logp.float(), (adv >= 0) | (w == 0)))
    free, kept = ratio * adv, ratio.clamp(1 - clip_low, 1 + clip_high) * adv
    clipped = kept < free
    per = -torch.where(clipped, kept.detach(), free)
    kl = zero
    if ref_logp is not None:
        u = finite(ref_logp.float() - logp, w == 0)
        kl = torch.expm1(u) - u
        if kl_coef != 0:
            per = per + kl_coef * kl
    per = torch.where(counts, per, zero)
    return (w * per).sum(), torch.stack([(w * kl).sum(), (w * clipped).sum()]).detach()


def preference_loss_plain(logp, targets, ref_logp, beta, label_smoothing):
    """(loss, rewards) of ``ops.kernels.preference_loss`` from log-probabilities [2P, T], by autograd in them alone."""
    counts = targets != IGNORE
    diff = logp if ref_logp is None else logp - ref_logp.detach().float()
    rewards = beta * torch.where(counts, diff, torch.zeros_like(diff)).sum(1, dtype=torch.float64).view(2, -1)
    z = rewards[0] - rewards[1]
    loss = -(1 - label_smoothing) * F.logsigmoid(z) - label_smoothing * F.logsigmoid(-z)
    return loss.mean().float(), rewards.detach().float()


# ---- entry points ----------------------------------------------------------------------
def token_logprobs(model, idx: torch.Tensor, targets: torch.Tensor, return_aux: bool = False):
    """Log-probability of ``targets`` [B, T] at every position: fp32 [B, T], differentiable, 0 where the target is -100.

    ``return_aux``: (log-probabilities, aux loss). A mixture-of-experts model that trains on a loss built from them adds
    the aux loss to it, as the other objectives' callers do: without it the routers' load is not balanced."""
    _check(idx, targets)
    fused = _fused(model, idx)
    x, aux = _trunk(model, idx, fused)
    if fused:
        logp = _HeadLogp.apply(*_head_args(model, x, targets)).view(idx.shape)
    else:
        logp = _logp_plain(model, x, targets)
    return (logp, aux) if return_aux else logp


def policy_loss(model, idx: torch.Tensor, targets: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor,
                ref_logp: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0):
    """Clipped policy loss with a KL term (formula: ``ops.kernels.policy_loss``).

    Returns (loss, aux loss, stats [2], logp [B, T]).
    ``old_logp``, ``ref_logp`` and ``weights`` [B, T]; ``advantages`` [B, T], or [B]: one per sequence. Tokens whose
    target is -100 take no part. ``stats`` = (weighted KL to the reference, weighted share of clipped tokens).
    All but the model is constant: no gradient goes to ``old_logp``, ``advantages``, ``ref_logp`` or ``weights``."""
    _check(idx, targets, old_logp=old_logp, ref_logp=ref_logp, weights=weights)
    _check_policy(clip_low, clip_high, kl_coef)
    if advantages.shape != idx.shape and advantages.shape != idx.shape[:1]:
        raise ValueError(f"advantages must be [B, T] or [B], got {tuple(advantages.shape)}")
    fused = _fused(model, idx)
    x, aux = _trunk(model, idx, fused)
    if fused:
        loss, stats, logp = _HeadPolicy.apply(
            *_head_args(model, x, targets), _flat32(old_logp), _flat32(advantages), _flat32(ref_logp), _flat32(weights),
            clip_low, clip_high, kl_coef, getattr(model, "loss_grad_hint", 1.0),
            getattr(model, "loss_grad_scale", None))
        return loss, aux, stats, logp.view(idx.shape)
    logp = _logp_plain(model, x, targets)
    loss, stats = policy_loss_plain(logp, targets, old_logp, advantages, ref_logp, weights, clip_low, clip_high,
                                    kl_coef)
    return loss, aux, stats, logp.detach()


def preference_loss(model, idx: torch.Tensor, targets: torch.Tensor, ref_logp: Optional[torch.Tensor] = None,
                    beta: float = 0.1, label_smoothing: float = 0.0):
    """Preference loss on pairs (formula: ``ops.kernels.preference_loss``): (loss, aux loss, rewards [2, P]).

    ``idx`` and ``targets`` [2P, T]: P chosen sequences, then their P rejected partners; ``ref_logp`` [2P, T]: the
    reference model's ``token_logprobs`` on the same tokens, a constant (none: a reference-free loss)."""
    _check(idx, targets, ref_logp=ref_logp)
    _check_preference(beta, label_smoothing)
    if idx.shape[0] % 2:
        raise ValueError(f"a preference batch holds chosen and rejected halves, got {idx.shape[0]} sequences")
    fused = _fused(model, idx)
    x, aux = _trunk(model, idx, fused)
    if fused:
        logp = _HeadLogp.apply(*_head_args(model, x, targets)).view(idx.shape)
        ref = None if ref_logp is None else ref_logp.float().contiguous()
        loss, rewards = _Preference.apply(logp, targets.contiguous(), ref, beta, label_smoothing)
        return loss, aux, rewards
    loss, rewards = preference_loss_plain(_logp_plain(model, x, targets), targets, ref_logp, beta, label_smoothing)
    return loss, aux, rewards
