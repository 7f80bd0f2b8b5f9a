"""Definitions of the decoding operators in 64 bits, and the bounds of what 32-bit arithmetic may differ from them."""
import math

import torch


def act8_values(x):
    """What a cache in 8 bits keeps of x [..., D]: 2^e is the least power of two, e >= -126, with max|x| <= 127 * 2^e; values
    are multiples of it, ties to even; NaN where x holds an infinity or NaN. Also the exponent bytes."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    broken = ~torch.isfinite(x).all(-1, keepdim=True)
    top = torch.where(broken, 1.0, top)
    mant, ex = torch.frexp(top)
    e = torch.where(mant > 127 / 128, ex - 6, ex - 7).clamp_min(-126).double()
    e = torch.where(top == 0, -126.0, e)
    v = torch.round(x / torch.exp2(e)) * torch.exp2(e)
    byte = torch.where(broken, 255.0, e + 127)[..., 0].to(torch.uint8)
    return torch.where(broken, math.nan, v), byte


class Cache:
    """Pages of a cache that hold NaN (codes: 127 under an exponent byte of NaN) wherever nothing was written."""

    def __init__(self, pages, heads, size, dim, dtype, bits, device="cuda"):
        self.bits, self.dtype, self.size = bits, dtype, size
        shape = (pages, heads, size, dim)
        if bits == 8:
            self.pools = {n: torch.full(shape, 127, dtype=torch.int8, device=device) for n in ("k_pages", "v_pages")}
            self.pools |= {n: torch.full(shape[:3], 255, dtype=torch.uint8, device=device) for n in ("k_exp", "v_exp")}
        else:
            self.pools = {n: torch.full(shape, math.nan, dtype=dtype, device=device) for n in ("k_pages", "v_pages")}

    def put(self, slots, k, v):
        """Writes K and V by indexing, from the format's definition."""
        page, at = slots // self.size, slots % self.size
        for n, x in (("k", k), ("v", v)):
            if self.bits == 8:
                val, byte = act8_values(x)
                scale = torch.exp2(byte.double() - 127)[..., None]
                self.pools[n + "_pages"][page, :, at] = (val / scale).nan_to_num(0).to(torch.int8)
                self.pools[n + "_exp"][page, :, at] = byte
            else:
                self.pools[n + "_pages"][page, :, at] = x

    def kept(self, x):
        return act8_values(x)[0] if self.bits == 8 else x.double()


def attention(q, k, v, scale):
    """One sequence: q [heads, D], k and v [tokens, kv heads, D] in 64 bits -> out [heads, D], lse [heads], and for the bound
    the largest sum |q k| scale of a head's scores and the mean |v| under its weights."""
    H, D = q.shape
    G = H // k.shape[1]
    k, v = (x.transpose(0, 1).repeat_interleave(G, 0) for x in (k, v))  # [heads, tokens, D]
    q = q.double()
    if k.shape[1] == 0:
        zero = torch.zeros_like(q)
        return zero, torch.full((H,), -math.inf, dtype=torch.float64, device=q.device), zero[:, 0], zero
    s = (k @ q[..., None])[..., 0] * scale
    lse = torch.logsumexp(s, 1)
    p = torch.exp(s - lse[:, None])
    size = (k.abs() @ q.abs()[..., None])[..., 0].amax(1) * abs(scale)
    return (p[:, None] @ v)[:, 0], lse, size, (p[:, None] @ v.abs())[:, 0]


def attention_bounds(out, lse, size, mean_v, D, n, dtype):
    """How far a result may be off whose scores, exponentials and sums are in 32 bits.

    A score is a sum of D exact products in 32 bits, in any order, times the scale and log2 e: off by at most
    (D + 2) 2^-24 size, and its difference to the maximum (at most 2 size) rounds by 2^-24 of it: ds <= (D + 6) 2^-24 size.
    A weight is off by the factor e^(2 ds) (its own score and the maximum), 2^-22 of the exponential, and what two 16-bit
    parts of bf16 (8 + 8 bits) leave of it, 2^-17; the sums of n weights and of n products, in chains of at most n,
    by n 2^-24 each at worst; partial results are joined by at most 3 more factors of 2^-22. Numerator and denominator each
    may be off by that. The output is rounded once: half a step of its type."""
    ds = (D + 6) * 2.0 ** -24 * size
    off = torch.expm1(2 * ds) + 2.0 ** -17 + 4 * 2.0 ** -22 + n * 2.0 ** -24
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return half * out.abs() + 2 * off[:, None] * (1 + half) * mean_v + tiny, ds + off + 2.0 ** -23 * lse.abs()


def sample_row(x, u, temperature, top_k, top_p, min_p):
    """The token of one row of logits (any device; computed in 64 bits on the CPU)."""
    x = x.double().cpu()
    V = x.numel()
    if any(math.isnan(s) for s in (u, temperature, top_p, min_p)) or bool((torch.isnan(x) | (x == math.inf)).any()):
        return -1
    top = float(x.max())
    if top == -math.inf:
        return -1
    x, order = torch.sort(x, descending=True, stable=True)
    if temperature <= 0 or top_p <= 0 or min_p > 1:
        return int(order[0])
    w = torch.where(x == -math.inf, 0.0, torch.where(x == top, 1.0, torch.exp((x - top) / temperature)))
    keep = torch.ones(V, dtype=torch.bool)
    if 0 < top_k < V:
        keep[top_k:] = False
    w = torch.where(keep, w, 0.0)
    if top_p < 1:
        keep &= (w.cumsum(0) - w) < top_p * w.sum()
    if min_p > 0 and temperature < math.inf:
        keep &= x >= top + temperature * math.log(min_p)
    keep[0] = True
    back = torch.zeros(V, dtype=torch.float64).scatter_(0, order, torch.where(keep, w, 0.0))
    run = back.cumsum(0)
    target = min(max(u, 0.0) * float(run[-1]), float(run[-1]))
    past = (run > target).nonzero()[:, 0]
    return int(past[0]) if past.numel() else int(back.nonzero()[-1])
