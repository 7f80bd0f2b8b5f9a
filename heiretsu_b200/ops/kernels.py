"""Thin Python wrappers over the extension's non-GEMM kernels.

Every wrapper allocates its outputs (unless given) with the PyTorch caching
allocator on the current stream and launches exactly one sm_100a kernel
sequence; nothing here falls back to a PyTorch implementation.
"""
from __future__ import annotations

from typing import Optional

import torch

from ._C import load


def _ext():
    return load()


# ---------------------------------------------------------------------------
# LayerNorm
# ---------------------------------------------------------------------------
def layernorm_fwd(x: torch.Tensor, w: torch.Tensor, b: torch.Tensor, eps: float = 1e-5,
                  dtype: torch.dtype = torch.bfloat16):
    """fp32 x [M, H] -> (y [M, H] in the 16-bit ``dtype`` (bf16 or fp16), mean [M], rstd [M])."""
    M = x.numel() // x.shape[-1]
    y = torch.empty(x.shape, device=x.device, dtype=dtype)
    mean = torch.empty(M, device=x.device, dtype=torch.float32)
    rstd = torch.empty(M, device=x.device, dtype=torch.float32)
    _ext().layernorm_fwd(x, w, b, y, mean, rstd, eps)
    return y, mean, rstd


def layernorm_bwd(dy, x, mean, rstd, w, dres_in, dres, dres16, dgamma, dbeta, scratch=None, dy_srcs: int = 1):
    """dres = dres_in + dLN/dx(dy); dres16 = 16-bit(dres); dgamma/dbeta (fp32) += partials.

    With ``dy_srcs > 1`` the output gradient is the sum of that many [M, H]
    slots of ``dy`` (the receive buffer of a reduce-scatter)."""
    H = x.shape[-1]
    M = x.numel() // H
    if scratch is None:
        rows = _ext().layernorm_bwd_scratch_rows(M)
        scratch = torch.empty(rows * 2 * H, device=x.device, dtype=torch.float32)
    _ext().layernorm_bwd(dy, x, mean, rstd, w, dres_in, dres, dres16, scratch, dgamma, dbeta, dy_srcs)


def resid_sum_ln(x, parts, nsrc, bias, x_new, w=None, b=None, y=None, mean=None, rstd=None, eps: float = 1e-5):
    """x_new = x + sum of `nsrc` 16-bit partial slots + bias; optionally y = LN(x_new) (16-bit, the slots' format)."""
    _ext().resid_sum_ln(x, parts, nsrc, bias, x_new, w, b, y, mean, rstd, eps)


def colsum_bf16(x: torch.Tensor, out: torch.Tensor) -> None:
    """out (fp32) += column sums of 16-bit (bf16 or fp16) x [M, N]."""
    _ext().colsum_bf16(x, out)


# ---------------------------------------------------------------------------
# Cross-entropy
# ---------------------------------------------------------------------------
def cross_entropy_fwd(logits: torch.Tensor, V: int, targets: torch.Tensor, ignore_index: int = -100):
    """16-bit logits [M, Vp] -> (mean loss (0-d fp32), lse [M], per-row loss [M])."""
    M = logits.shape[0]
    lse = torch.empty(M, device=logits.device, dtype=torch.float32)
    rows = torch.empty(M, device=logits.device, dtype=torch.float32)
    mean = torch.empty((), device=logits.device, dtype=torch.float32)
    _ext().cross_entropy_fwd(logits, V, targets, ignore_index, lse, rows, mean)
    return mean, lse, rows


def cross_entropy_fused_(logits: torch.Tensor, V: int, targets: torch.Tensor, scale: torch.Tensor,
                         ignore_index: int = -100):
    """Forward and gradient in one pass: returns (mean loss, lse) and leaves
    (softmax - onehot) * scale in ``logits`` (columns >= V zeroed); ``scale`` fp32 [1]."""
    M = logits.shape[0]
    lse = torch.empty(M, device=logits.device, dtype=torch.float32)
    rows = torch.empty(M, device=logits.device, dtype=torch.float32)
    mean = torch.empty((), device=logits.device, dtype=torch.float32)
    _ext().cross_entropy_fused(logits, V, targets, ignore_index, lse, rows, mean, scale)
    return mean, lse


def cross_entropy_rescale_(g: torch.Tensor, actual: torch.Tensor, expected: torch.Tensor) -> torch.Tensor:
    """In place g *= actual / expected (fp32 [1] device scalars); nothing happens when equal."""
    _ext().cross_entropy_rescale(g, actual, expected)
    return g


def cross_entropy_bwd_(logits, V, targets, lse, scale: Optional[torch.Tensor], scale_mul: float,
                       ignore_index: int = -100) -> torch.Tensor:
    """In place: logits <- (softmax - onehot) * scale * scale_mul (columns >= V zeroed)."""
    _ext().cross_entropy_bwd(logits, V, targets, ignore_index, lse, scale, scale_mul)
    return logits


# ---------------------------------------------------------------------------
# Post-training losses (the outputs of these and of the 8-bit activations are allocated by
# the extension: that halves the host's share of a short call)
# ---------------------------------------------------------------------------
def token_logprobs(logits: torch.Tensor, V: int, targets: torch.Tensor, ignore_index: int = -100,
                   grad: Optional[torch.Tensor] = None):
    """Log-probability of each row's target token: (logp [M], lse [M]), fp32.

    ``logits`` [M, >= V] in bf16, fp16 or fp32 with contiguous rows (any row stride, any alignment), ``targets``
    int64 [M]. Rows whose target is ``ignore_index`` give 0 in both, whatever they hold; a target outside [0, V) gives
    NaN and the bad-argument status. V is limited by shared memory (about 920,000 in 16 bits, 460,000 in fp32).
    Equal logits (and shapes) give equal bits here, with ``grad``, and in ``policy_loss``. ``grad`` (a buffer like
    ``logits``, or ``logits`` itself: in place) receives the gradient of each row's log-probability, onehot - softmax,
    zero in ignored rows and in columns >= V: the gradient of any loss of the log-probabilities is this with row i
    times dloss/dlogp[i]."""
    return _ext().token_logprobs(logits, V, targets, ignore_index, grad)


def policy_loss(logits: torch.Tensor, V: int, targets: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor,
                ref_logp: Optional[torch.Tensor] = None, weights: Optional[torch.Tensor] = None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, grad_scale: Optional[torch.Tensor] = None,
                ignore_index: int = -100, grad: Optional[torch.Tensor] = None):
    """Clipped policy loss with a KL term, and its gradient in the logits, in one pass over them.

    Per counted row, with logp as in ``token_logprobs``, r = exp(logp - old_logp), A the advantage, u = ref_logp - logp:
    l = -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (e^u - u - 1). The loss is sum w l with w =
    ``weights`` [M], or one over the number of counted rows. ``advantages`` fp32: [M], or one value for each of n
    equal runs of rows (M % n == 0: a value per sequence). Returns (loss (0-d), stats [2] = (sum w KL, sum w over
    clipped rows), logp [M], grad): ``grad`` (a new tensor like ``logits``, the given buffer, or ``logits`` itself)
    is the loss's gradient times the device scalar ``grad_scale`` (fp32 [1], default 1). Without ``ref_logp``
    there is no KL term and its statistic is 0."""
    return _ext().policy_loss(logits, V, targets, old_logp, advantages, ref_logp, weights, clip_low, clip_high, kl_coef,
                              grad_scale, ignore_index, grad)


def preference_loss(logp: torch.Tensor, targets: torch.Tensor, ref_logp: Optional[torch.Tensor] = None,
                    beta: float = 0.1, label_smoothing: float = 0.0, ignore_index: int = -100):
    """Paired log-ratio loss of token log-probabilities and its gradient: (loss (0-d), rewards [2, P], dlogp [2P, T]).

    ``logp`` fp32 [2P, T]: P chosen sequences, then their P rejected partners; tokens whose target is ``ignore_index``
    take no part (a sequence without any counts 0). With S = sum over a sequence of logp - ref_logp (``ref_logp``
    like ``logp``; none: 0), rewards = beta S and z = beta (S_chosen - S_rejected), the loss is the mean over pairs of
    -(1 - label_smoothing) log sigmoid(z) - label_smoothing log sigmoid(-z); sums run in 64 bits."""
    return _ext().preference_loss(logp, targets, ref_logp, beta, label_smoothing, ignore_index)


# ---------------------------------------------------------------------------
# Activations in 8 bits (format: csrc/act8.cuh)
# ---------------------------------------------------------------------------
def act8_pack(x: torch.Tensor):
    """x [M, N] (bf16, fp16 or fp32, contiguous rows) -> (q int8 [M, N], e uint8 [M, ceil(N / 128)]).

    A block of 128 columns keeps 2^(e - 127), the least power of two >= max|x| / 127 (and >= 2^-126), and codes
    x / 2^(e - 127) rounded to nearest even: each value is off by at most max|x| / 127 of its block. A block with an
    infinity or NaN comes back as NaN."""
    return _ext().act8_pack(x)


def act8_unpack(q: torch.Tensor, e: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of ``act8_pack``'s codes in bf16, fp16 or fp32 (clamped to the type's largest finite value)."""
    return _ext().act8_unpack(q, e, dtype, False)[0]


def act8_unpack_gelu(q: torch.Tensor, e: torch.Tensor, dtype: torch.dtype = torch.bfloat16):
    """(GELU(x), x) with x = ``act8_unpack(q, e, dtype)``: both operands of the MLP's backward from its kept
    pre-activation (tanh form of GELU, evaluated on the unrounded value)."""
    x, h = _ext().act8_unpack(q, e, dtype, True)
    return h, x


def layernorm_fwd_act8(x: torch.Tensor, w: torch.Tensor, b: torch.Tensor, eps: float = 1e-5,
                       dtype: torch.dtype = torch.bfloat16):
    """``layernorm_fwd`` that keeps xh = (x - mean) rstd in 8 bits instead of x, mean and y for the backward:
    fp32 x [M, H] -> (y in the 16-bit ``dtype``, q, e, rstd [M])."""
    return _ext().layernorm_fwd_act8(x, w, b, eps, dtype)


def layernorm_bwd_act8(dy, q, e, rstd, w, b, dres_in, dres, dres16, dgamma, dbeta) -> torch.Tensor:
    """``layernorm_bwd`` from the kept codes: dres = dres_in + dLN/dx(dy) (``dres`` may be ``dres_in``), dres16 =
    16-bit(dres), dgamma / dbeta (fp32) += their sums. Returns y = xh w + b of the kept xh in dres16's format: the
    operand of the next weight gradient."""
    return _ext().layernorm_bwd_act8(dy, q, e, rstd, w, b, dres_in, dres, dres16, dgamma, dbeta)


# ---------------------------------------------------------------------------
# Decoding: a paged key/value cache, attention of one new token over it, and the choice of the next token
# ---------------------------------------------------------------------------
# A cache is k_pages and v_pages [pages, heads, page size, head dim] (bf16 or fp16; the page size a multiple of 16, any
# strides that are multiples of 16 bytes). In 8 bits they are int8 and k_exp and v_exp (uint8 [pages, heads, page size]) hold
# the exponent byte of each head of each token: the format of act8_pack with a block per head of a token.
def kv_write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
             k_exp: Optional[torch.Tensor] = None, v_exp: Optional[torch.Tensor] = None) -> None:
    """Writes K and V of new tokens ([tokens, heads, head dim], bf16 or fp16; any strides, such as views of a projection's
    output) into the cache, quantised where it holds 8 bits.

    ``slots`` int64 [tokens]: page * page size + place in the page. A negative slot's token is not kept; one behind the
    cache is not either, and sets the bad-argument status. Slots must differ: of two tokens with one slot either may be kept,
    or a mixture of both. An 8-bit head that holds an infinity or NaN comes back as NaN."""
    _ext().kv_write(k, v, slots, k_pages, v_pages, k_exp, v_exp)


def kv_read(slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, k_exp: Optional[torch.Tensor] = None,
            v_exp: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None):
    """K and V of ``slots`` (as in ``kv_write``; the same slot may come more than once): (k, v) [tokens, heads, head dim].

    An 8-bit cache is read in ``dtype`` (bf16, the default, fp16 or fp32; values beyond the type's range become its
    largest), a 16-bit one in its own. A negative slot reads as zeros; one behind the cache as NaN, and sets the
    bad-argument status."""
    return _ext().kv_read(slots, k_pages, v_pages, k_exp, v_exp, dtype)


def decode_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                     lengths: torch.Tensor, k_exp: Optional[torch.Tensor] = None, v_exp: Optional[torch.Tensor] = None,
                     scale: Optional[float] = None):
    """Attention of one new token per sequence over its cached tokens: (out like q, lse fp32 [sequences, heads]).

    ``q`` [sequences, heads, head dim] in bf16 or fp16 (any strides; a 16-bit cache has its dtype), heads a multiple of
    the cache's: query heads i * g .. i * g + g - 1 share K/V head i. ``table`` int32 [sequences, pages]: the pages of a
    sequence in order; ``lengths`` int32 [sequences]: how many of its tokens count, the new one's own K and V among them when
    it has been written. Entries and slots behind them are not read. ``scale`` defaults to head dim ** -0.5; ``lse`` is the natural
    log-sum-exp of the scores, so that outputs over parts of a cache can be joined. A sequence of length 0 gives 0 and
    -inf; a length or page out of range gives NaN in its rows, and sets the bad-argument status. A NaN or infinity in a counted
    token's V makes its channel NaN, in its K the row (-inf scores weigh nothing)."""
    return _ext().decode_attention(q, k_pages, v_pages, table, lengths, k_exp, v_exp, scale)


def _per_row(value):
    """A setting of ``sample_tokens`` as (tensor or None, number)."""
    return (value, 0) if isinstance(value, torch.Tensor) else (None, value)


def sample_tokens(logits: torch.Tensor, V: int, u: torch.Tensor, temperature=1.0, top_k=0, top_p=1.0,
                  min_p=0.0) -> torch.Tensor:
    """A token per row of ``logits`` [M, >= V] (bf16, fp16 or fp32, contiguous rows): int64 [M].

    ``u`` fp32 [M]: uniform numbers in [0, 1). Settings are numbers, or tensors [M] with one for each row (fp32; ``top_k``
    int64). Token i weighs w_i = exp((x_i - max) / temperature). In the order by logit, descending, equal ones by index, kept
    are the first ``top_k`` (0, or V and more: all), of these the shortest start whose weight reaches ``top_p`` of theirs, of
    these the ones with w_i >= ``min_p``; the first always is. The token drawn is the first kept one, in the
    vocabulary's order, at which the running weight exceeds u times the kept weight: the same u, logits and settings
    give the same token whatever the other rows are. ``temperature`` <= 0 takes the largest logit (equal ones: the lowest
    index). A row that holds +inf or NaN, or nothing but -inf, and a setting or u that is NaN, gives -1. V is at most 524288."""
    t, t0 = _per_row(temperature)
    k, k0 = _per_row(top_k)
    p, p0 = _per_row(top_p)
    m, m0 = _per_row(min_p)
    return _ext().sample_tokens(logits, V, u, t, float(t0), k, int(k0), p, float(p0), m, float(m0))


# ---------------------------------------------------------------------------
# Embedding
# ---------------------------------------------------------------------------
def embedding_fwd(idx: torch.Tensor, wte: torch.Tensor, wpe: torch.Tensor) -> torch.Tensor:
    B, T = idx.shape
    out = torch.empty(B * T, wte.shape[1], device=idx.device, dtype=torch.float32)
    _ext().embedding_fwd(idx, wte, wpe, out)
    return out


def embedding_bwd(idx, dx, dwte: Optional[torch.Tensor], dwpe: Optional[torch.Tensor]) -> None:
    _ext().embedding_bwd(idx, dx, dwte, dwpe)


# ---------------------------------------------------------------------------
# Optimizer pieces
# ---------------------------------------------------------------------------
def sumsq(x: torch.Tensor, out: torch.Tensor, weight: float = 1.0, accumulate: bool = False, scratch=None):
    """out (0-d fp32) (+)= weight * sum(x^2), deterministic two-pass."""
    if scratch is None:
        scratch = torch.empty(_ext().sumsq_scratch_size(), device=x.device, dtype=torch.float32)
    _ext().sumsq(x, scratch, weight, out, accumulate)


def clip_coef(norm2: torch.Tensor, max_norm: float, coef: torch.Tensor, norm: Optional[torch.Tensor] = None,
              loss_scale: Optional[torch.Tensor] = None):
    """coef = min(1, max_norm / norm) (NaN when the norm is not finite). With ``loss_scale``
    (fp32 device scalar S) the gradients hold S * g: the norm is unscaled and coef carries 1/S."""
    _ext().clip_coef(norm2, max_norm, coef, norm, loss_scale)


def loss_scale_update(coef: torch.Tensor, state: torch.Tensor, growth: float = 2.0, backoff: float = 0.5,
                      interval: int = 2000) -> None:
    """Dynamic loss scale on the device: state = [scale, finite steps in a row] (fp32)."""
    _ext().loss_scale_update(coef, state, growth, backoff, interval)


def adamw_step(p, grad, m, v, p16, hyper, coef=None):
    _ext().adamw_step(p, grad, m, v, p16, hyper, coef)


def f32_to_bf16(x: torch.Tensor, y: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """fp32 -> 16-bit copy (into ``y``, else a new tensor of ``dtype``: bf16 or fp16)."""
    if y is None:
        y = torch.empty(x.shape, device=x.device, dtype=dtype)
    _ext().f32_to_bf16(x, y)
    return y


# ---------------------------------------------------------------------------
# Attention (causal; head_dim 16, 32, 64 or 128)
# ---------------------------------------------------------------------------
def attention_fwd(qkv: torch.Tensor, B: int, T: int, nh: int, out: Optional[torch.Tensor] = None, drop=None,
                  head_dim: int = 64):
    """qkv [B*T, 3*nh*dh] (bf16 or fp16) -> (y [B*T, nh*dh] same format, nlse fp32 [B, nh, Tpad]), dh = head_dim.

    nlse = -log2(sum_k 2^(s_k * log2(e) / sqrt(dh))) per query row: the negated
    log2-domain log-sum-exp, kept in the form the backward kernel consumes.
    Natural-log LSE = -nlse * ln(2).

    ``drop = (seed_tensor, site, p, h0, nh_total)`` applies dropout to the
    attention probabilities (mask of heads h0 .. h0+nh-1 of nh_total; see
    ops/dropout_ref.py); the backward must get the same ``drop``."""
    Tpad = (T + 127) // 128 * 128
    if out is None:
        out = torch.empty(B * T, nh * head_dim, device=qkv.device, dtype=qkv.dtype)
    lse = torch.empty(B, nh, Tpad, device=qkv.device, dtype=torch.float32)
    d_seed, d_site, d_p, h0, nht = drop if drop is not None else (None, 0, 0.0, 0, 0)
    _ext().attention_fwd(qkv, B, T, nh, out, lse, d_seed, int(d_site), float(d_p), int(h0), int(nht), int(head_dim))
    return out, lse


def attention_bwd(qkv, out, dout, lse, B, T, nh, dqkv: Optional[torch.Tensor] = None, drop=None,
                  head_dim: int = 64):
    """Returns dqkv [B*T, 3*nh*dh] in qkv's format (columns [dQ | dK | dV])."""
    Tpad = (T + 127) // 128 * 128
    if dqkv is None:
        dqkv = torch.empty(B * T, 3 * nh * head_dim, device=qkv.device, dtype=qkv.dtype)
    dvec = torch.empty(B, nh, Tpad, device=qkv.device, dtype=torch.float32)
    dq_acc = torch.empty(B * T, nh * max(head_dim, 64), device=qkv.device, dtype=torch.float32)
    d_seed, d_site, d_p, h0, nht = drop if drop is not None else (None, 0, 0.0, 0, 0)
    _ext().attention_bwd(qkv, out, dout, lse, B, T, nh, dvec, dq_acc, dqkv, d_seed, int(d_site), float(d_p), int(h0),
                         int(nht), int(head_dim))
    return dqkv


def dropout_bf16(g: torch.Tensor, seed: torch.Tensor, site: int, p: float, row0: int = 0,
                 out: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """16-bit(g * mask) for residual dropout site ``site`` (g fp32 [M, H]; out bf16 or fp16)."""
    if out is None:
        out = torch.empty(g.shape, device=g.device, dtype=dtype)
    _ext().dropout_bf16(g, out, seed, int(site), float(p), int(row0))
    return out
