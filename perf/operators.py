"""Post-training losses on the vocabulary logits, and activations kept in 8 bits: plain forms, kernels, and the cases they are timed on.

Operators (``case["op"]``):

* ``logprobs``    log-probability of each row's target token (and, with ``grad``, its gradient in the logits)
* ``policy``      clipped policy loss with a KL term on the logits: loss, statistics, log-probabilities, gradient
* ``preference``  paired log-ratio loss on token log-probabilities: loss, rewards, gradient
* ``act8``        an activation packed into 8 bits (a power-of-two scale per 128 columns) and restored for backward
* ``norm8``       LayerNorm that keeps its normalised input in 8 bits: forward, and the backward that reads it

``run`` computes the plain form (elementary torch operations) while ``own`` is false and calls the framework's
kernels (``heiretsu_b200.ops.kernels``) while it is true.
"""
import math

import torch

own = False

IGNORE = -100  # targets with this value take no part (prompt and padding tokens)
BLOCK = 128    # columns that share one scale in the 8-bit format
EPS = 1e-5     # LayerNorm
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BETA, SMOOTHING = 0.1, 0.05
CLIP_LOW, CLIP_HIGH, KL_COEF = 0.2, 0.28, 0.04


def listed():
    return [
        # one decoding step of 16 sequences: score the tokens just sampled (latency)
        {"name": "logprobs step 16", "op": "logprobs", "rows": 16, "vocab": 50257, "type": "bf16", "pad": True, "grad": False},
        # the frozen reference model scores a micro-batch of 8 x 1024 tokens
        {"name": "logprobs reference 8k", "op": "logprobs", "rows": 8192, "vocab": 50257, "type": "bf16", "pad": True, "grad": False},
        # the trained model scores 4 x 1024 tokens and keeps the gradient, fp16 training
        {"name": "logprobs grad fp16 4k", "op": "logprobs", "rows": 4096, "vocab": 50257, "type": "fp16", "pad": True, "grad": True},
        # one short sampled answer (61 tokens), with the KL term
        {"name": "policy answer 61", "op": "policy", "rows": 61, "vocab": 50257, "type": "bf16", "pad": True, "ref": True, "weights": True},
        # a policy step on a micro-batch of 8 x 1024 tokens, with the KL term
        {"name": "policy batch 8k", "op": "policy", "rows": 8192, "vocab": 50257, "type": "bf16", "pad": True, "ref": True, "weights": False},
        # fp32 logits of an odd, unpadded vocabulary (rows that start on 4-byte boundaries only)
        {"name": "policy fp32 odd 500", "op": "policy", "rows": 500, "vocab": 32003, "type": "fp32", "pad": False, "ref": False, "weights": False},
        # a single short pair
        {"name": "preference pair 57", "op": "preference", "pairs": 1, "length": 57, "ref": False},
        # 64 pairs of up to 1024 tokens against the reference model
        {"name": "preference batch 64x1k", "op": "preference", "pairs": 64, "length": 1024, "ref": True},
        # a block's input (fp32 residual stream) of 8 x 1024 tokens at GPT-2 large's width, kept for recomputation
        {"name": "act8 residual 8k", "op": "act8", "rows": 8192, "cols": 1280, "type": "fp32", "gelu": False},
        # the MLP pre-activation of 8 x 1024 tokens at GPT-2 large's width: kept, then restored with its GELU
        {"name": "act8 gelu 8k", "op": "act8", "rows": 8192, "cols": 5120, "type": "bf16", "gelu": True},
        # forward of a short odd batch at GPT-2 small's width, fp16
        {"name": "norm8 forward 1000", "op": "norm8", "rows": 1000, "cols": 768, "type": "fp16", "back": False},
        # backward of 8 x 1024 tokens at GPT-2 large's width
        {"name": "norm8 backward 8k", "op": "norm8", "rows": 8192, "cols": 1280, "type": "bf16", "back": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "policy", "preference", "act8", "norm8"])
    if op in ("logprobs", "policy"):
        kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        vocab = _log(rng, 1000, 130000)
        most = 8192 * 50257 * 2 // (vocab * (4 if kind == "fp32" else 2))
        case = {"op": op, "rows": _log(rng, 1, min(most, 8192)), "vocab": vocab, "type": kind, "pad": rng.random() < 0.7}
        if op == "logprobs":
            case["grad"] = rng.random() < 0.5
        else:
            case["ref"], case["weights"] = rng.random() < 0.7, rng.random() < 0.3
        return case
    if op == "preference":
        length = _log(rng, 1, 4096)
        return {"op": op, "pairs": _log(rng, 1, max(1, min(256, 131072 // length))), "length": length, "ref": rng.random() < 0.7}
    if op == "act8":
        cols = _log(rng, 16, 8192)
        return {"op": op, "rows": _log(rng, 1, 8192 * 5120 // cols if cols > 512 else 65536), "cols": cols,
                "type": rng.choice(["bf16", "fp16", "fp32"]), "gelu": rng.random() < 0.5}
    return {"op": op, "rows": _log(rng, 1, 16384), "cols": 4 * _log(rng, 8, 512), "type": rng.choice(["bf16", "fp16"]),
            "back": rng.random() < 0.5}


def _width(case):
    return (case["vocab"] + 127) // 128 * 128 if case["pad"] else case["vocab"]


# ---- inputs ----------------------------------------------------------------------
def _logits(case, g):
    """Logits of a trained model: normal, with the target token raised by 4 to 14."""
    M, V, W, dt = case["rows"], case["vocab"], _width(case), TYPES[case["type"]]
    logits = torch.zeros(M, W, device="cuda", dtype=dt)
    targets = torch.randint(0, V, (M,), device="cuda", generator=g)
    for a in range(0, M, 1024):
        b = min(M, a + 1024)
        x = torch.randn(b - a, V, device="cuda", generator=g).mul_(2.0)
        x.scatter_add_(1, targets[a:b, None], 4 + 10 * torch.rand(b - a, 1, device="cuda", generator=g))
        logits[a:b, :V] = x
    return logits, targets


def _logp64(logits, V, targets):
    out = torch.empty(logits.shape[0], device="cuda", dtype=torch.float64)
    for a in range(0, logits.shape[0], 512):
        x = logits[a:a + 512, :V].double()
        out[a:a + 512] = x.gather(1, targets[a:a + 512, None].clamp_min(0))[:, 0] - torch.logsumexp(x, 1)
    return out


def _spans(n, length, g):
    """[n, length] truth values of the answer tokens: a prompt of up to a half before them, padding behind."""
    at = torch.arange(length, device="cuda")[None]
    first = (torch.rand(n, 1, device="cuda", generator=g) * length * 0.5).long()
    last = first + 1 + (torch.rand(n, 1, device="cuda", generator=g) * (length - first)).long()
    return (at >= first) & (at < last)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], {"case": case}
    if op in ("logprobs", "policy"):
        s["logits"], s["targets"] = _logits(case, g)
        M = case["rows"]
        if op == "policy":
            # log-ratios of a run with stale samples: most tokens inside the clip range, some far outside
            now = _logp64(s["logits"], case["vocab"], s["targets"])
            far = torch.rand(M, device="cuda", generator=g) < 0.15
            side = torch.where(torch.rand(M, device="cuda", generator=g) < 0.5, -1.0, 1.0)
            wide = side * (0.35 + 0.3 * torch.rand(M, device="cuda", generator=g))
            near = (0.04 * torch.randn(M, device="cuda", generator=g)).clamp_(-0.15, 0.15)
            s["old"] = (now - torch.where(far, wide, near)).float()
            s["adv"] = torch.randn(M, device="cuda", generator=g)
            s["ref"] = (now + 0.3 * torch.randn(M, device="cuda", generator=g)).float() if case["ref"] else None
        # prompt and padding tokens take no part; one row at least does
        drop = torch.rand(M, device="cuda", generator=g) < 0.25
        drop[M // 2] = False
        s["targets"][drop] = IGNORE
        if op == "policy":
            s["weights"] = None
            if case["weights"]:  # each token weighs one over its answer's length
                s["weights"] = (0.5 + torch.rand(M, device="cuda", generator=g)) / M
    elif op == "preference":
        n, T = 2 * case["pairs"], case["length"]
        s["targets"] = torch.randint(0, 50257, (n, T), device="cuda", generator=g)
        s["targets"][~_spans(n, T, g)] = IGNORE
        counts = s["targets"] != IGNORE
        s["logp"] = -torch.empty(n, T, device="cuda").exponential_(0.5, generator=g) * counts
        s["ref"] = (s["logp"] + 0.2 * torch.randn(n, T, device="cuda", generator=g)) * counts if case["ref"] else None
    elif op == "act8":
        x = torch.randn(case["rows"], case["cols"], device="cuda", generator=g)
        x *= 0.2 + 2 * torch.rand(1, case["cols"], device="cuda", generator=g)  # channels of unlike sizes
        s["x"] = x.to(TYPES[case["type"]])
    else:
        M, H = case["rows"], case["cols"]
        x = torch.randn(M, H, device="cuda", generator=g) * (0.5 + torch.rand(1, H, device="cuda", generator=g)) + 0.1
        s["w"] = 1 + 0.1 * torch.randn(H, device="cuda", generator=g)
        s["b"] = 0.1 * torch.randn(H, device="cuda", generator=g)
        if not case["back"]:
            s["x"] = x
        else:
            mu = x.double().mean(1, keepdim=True)
            rstd = torch.rsqrt((x.double() - mu).square().mean(1, keepdim=True) + EPS)
            s["q"], s["e"] = _pack(((x - mu) * rstd).float())
            s["rstd"] = rstd[:, 0].float()
            s["dy"] = torch.randn(M, H, device="cuda", generator=g)
            s["dres_in"] = torch.randn(M, H, device="cuda", generator=g)
            s["dres"] = torch.empty_like(s["dres_in"])
            s["dres16"] = torch.empty(M, H, device="cuda", dtype=TYPES[case["type"]])
    return s


# ---- plain forms -----------------------------------------------------------------
def _pack(x):
    """x [M, N] -> codes int8 [M, N] and exponent bytes uint8 [M, ceil(N / 128)].

    e is the least whole number >= -126 with max|x| <= 127 * 2^e over the block (stored as e + 127); the code is
    x / 2^e rounded to the nearest whole number, ties to even. Scaling by a power of two is exact."""
    M, N = x.shape
    nb = (N + BLOCK - 1) // BLOCK
    xb = torch.nn.functional.pad(x.float(), (0, nb * BLOCK - N)).view(M, nb, BLOCK)
    mant, ex = torch.frexp(xb.abs().amax(2))  # max|x| = mant * 2^ex, mant in [0.5, 1)
    e = torch.where(mant * 128 > 127, ex - 6, ex - 7).clamp_min_(-126)
    e = torch.where(mant == 0, torch.full_like(e, -126), e)
    q = torch.ldexp(xb, -e[:, :, None].float()).round()
    return q.view(M, nb * BLOCK)[:, :N].to(torch.int8), (e + 127).to(torch.uint8)


def _unpack(q, e):
    scale = torch.ldexp(torch.ones((), device=q.device), e.float() - 127)
    return q.float() * scale.repeat_interleave(BLOCK, 1)[:, : q.shape[1]]


def _gelu(x):
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))


def _rows(logits, V, targets):
    """fp32 logits, log-sum-exp, target log-probability (0 where ignored) and the mask of rows that count."""
    x = logits[:, :V].float()
    top = x.amax(1, keepdim=True)
    lse = top + (x - top).exp().sum(1, keepdim=True).log()
    counts = targets != IGNORE
    logp = torch.where(counts, (x.gather(1, targets.clamp_min(0)[:, None]) - lse)[:, 0], 0.0)
    return x, lse, logp, counts


def _grad(x, lse, targets, coef, like):
    """coef * (onehot - softmax), columns behind the vocabulary zero, in like's type."""
    g = (x - lse).exp_().mul_(-coef[:, None])
    g.scatter_add_(1, targets.clamp_min(0)[:, None], coef[:, None])
    out = torch.zeros_like(like)
    out[:, : x.shape[1]] = g
    return out


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op in ("logprobs", "policy"):
        x, lse, logp, counts = _rows(s["logits"], case["vocab"], s["targets"])
        if op == "logprobs":
            if not case["grad"]:
                return {"logp": logp, "lse": torch.where(counts, lse[:, 0], 0.0)}
            return {"logp": logp, "lse": torch.where(counts, lse[:, 0], 0.0), "grad": _grad(x, lse, s["targets"], counts.float(), s["logits"])}
        w = counts.double() / counts.sum().clamp_min(1) if s["weights"] is None else s["weights"].double() * counts
        delta = torch.where(counts, logp.double() - s["old"], 0.0)
        ratio, adv = delta.exp(), s["adv"].double()
        kept = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
        clipped = kept * adv < ratio * adv
        loss = -torch.minimum(ratio * adv, kept * adv)
        coef = torch.where(clipped, 0.0, -ratio * adv)
        kl = torch.zeros_like(loss)
        if s["ref"] is not None:
            d = torch.where(counts, s["ref"].double() - logp, 0.0)
            kl = torch.expm1(d) - d
            loss, coef = loss + KL_COEF * kl, coef - KL_COEF * torch.expm1(d)
        stats = torch.stack([(w * kl).sum(), (w * clipped).sum()]).float()
        coef = torch.where(counts, w * coef, 0.0).float()
        return {"loss": (w * loss).sum().float(), "stats": stats, "logp": logp, "grad": _grad(x, lse, s["targets"], coef, s["logits"])}
    if op == "preference":
        P, counts = case["pairs"], s["targets"] != IGNORE
        diff = s["logp"].double() if s["ref"] is None else s["logp"].double() - s["ref"]
        reward = BETA * torch.where(counts, diff, 0.0).sum(1).view(2, P)
        z = reward[0] - reward[1]
        soft = lambda t: t.clamp_min(0) + torch.log1p(torch.exp(-t.abs()))  # noqa: E731  log(1 + e^t)
        loss = ((1 - SMOOTHING) * soft(-z) + SMOOTHING * soft(z)).mean()
        c = BETA / P * (SMOOTHING / (1 + torch.exp(-z)) - (1 - SMOOTHING) / (1 + torch.exp(z)))
        return {"loss": loss.float(), "rewards": reward.float(), "dlogp": (torch.cat([c, -c])[:, None] * counts).float()}
    if op == "act8":
        x = _unpack(*_pack(s["x"]))
        kept = x.to(s["x"].dtype)
        return {"x": kept, "gelu": _gelu(x).to(s["x"].dtype)} if case["gelu"] else {"x": kept}
    if not case["back"]:
        x = s["x"]
        mu = x.mean(1, keepdim=True)
        rstd = torch.rsqrt((x - mu).square().mean(1, keepdim=True) + EPS)
        xh = (x - mu) * rstd
        # the codes come back as the values they stand for (each fits 16 bits exactly)
        return {"y": (xh * s["w"] + s["b"]).to(TYPES[case["type"]]), "kept": _unpack(*_pack(xh)).bfloat16(), "rstd": rstd[:, 0]}
    xh, dy = _unpack(s["q"], s["e"]), s["dy"]
    gw = dy * s["w"]
    dx = s["rstd"][:, None] * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
    new = s["dres_in"] + dx
    half = TYPES[case["type"]]
    return {"dres": new, "dres16": new.to(half), "y": (xh * s["w"] + s["b"]).to(half),
            "dgamma": (dy * xh).double().sum(0).float(), "dbeta": dy.double().sum(0).float()}


# ---- the framework's calls ---------------------------------------------------------
def _calls(s):
    from heiretsu_b200.ops import kernels as K

    case = s["case"]
    op = case["op"]
    if op == "logprobs":
        if not case["grad"]:
            logp, lse = K.token_logprobs(s["logits"], case["vocab"], s["targets"])
            return {"logp": logp, "lse": lse}
        grad = torch.empty_like(s["logits"])
        logp, lse = K.token_logprobs(s["logits"], case["vocab"], s["targets"], grad=grad)
        return {"logp": logp, "lse": lse, "grad": grad}
    if op == "policy":
        loss, stats, logp, grad = K.policy_loss(s["logits"], case["vocab"], s["targets"], s["old"], s["adv"], ref_logp=s["ref"],
                                                weights=s["weights"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL_COEF)
        return {"loss": loss, "stats": stats, "logp": logp, "grad": grad}
    if op == "preference":
        loss, rewards, dlogp = K.preference_loss(s["logp"], s["targets"], ref_logp=s["ref"], beta=BETA, label_smoothing=SMOOTHING)
        return {"loss": loss, "rewards": rewards, "dlogp": dlogp}
    if op == "act8":
        q, e = K.act8_pack(s["x"])
        if case["gelu"]:
            h, x = K.act8_unpack_gelu(q, e, dtype=s["x"].dtype)
            return {"x": x, "gelu": h}
        return {"x": K.act8_unpack(q, e, dtype=s["x"].dtype)}
    if not case["back"]:
        y, q, e, rstd = K.layernorm_fwd_act8(s["x"], s["w"], s["b"], EPS, dtype=TYPES[case["type"]])
        return {"y": y, "kept": K.act8_unpack(q, e, dtype=torch.bfloat16), "rstd": rstd}
    dg, db = torch.zeros(2, case["cols"], device="cuda").unbind(0)
    y = K.layernorm_bwd_act8(s["dy"], s["q"], s["e"], s["rstd"], s["w"], s["b"], s["dres_in"], s["dres"], s["dres16"], dg, db)
    return {"dres": s["dres"], "dres16": s["dres16"], "y": y, "dgamma": dg, "dbeta": db}


def run(state):
    if own:
        return _calls(state)
    return _plain(state)


def work(case):
    """Bytes: every input read once and every output written once. Flops: one per elementary step of the formula."""
    op = case["op"]
    if op in ("logprobs", "policy"):
        M, V, W, es = case["rows"], case["vocab"], _width(case), 4 if case["type"] == "fp32" else 2
        if op == "logprobs":
            return {"bytes": M * (V * es + 16) + (M * W * es if case["grad"] else 0), "flops": M * V * (6 if case["grad"] else 3)}
        return {"bytes": M * (V * es + W * es + 8 + 12 + (4 if case["ref"] else 0) + (4 if case["weights"] else 0)), "flops": M * V * 6}
    if op == "preference":
        n = 2 * case["pairs"] * case["length"]
        return {"bytes": n * (8 + 4 + 4 + (4 if case["ref"] else 0)), "flops": n * 3}
    M, N = case["rows"], case["cols"]
    if op == "act8":  # packed in one call, restored in another: the codes cross memory twice
        es = 4 if case["type"] == "fp32" else 2
        return {"bytes": M * N * (es + 1 + 1 + es * (2 if case["gelu"] else 1)), "flops": M * N * (14 if case["gelu"] else 4)}
    if not case["back"]:  # x in; y, the codes, and the codes' values out
        return {"bytes": M * N * (4 + 2 + 1 + 1 + 2) + M * 4, "flops": M * N * 12}
    return {"bytes": M * N * (4 + 1 + 4 + 4 + 2 + 2) + M * 4 + N * 16, "flops": M * N * 14}


# ---- the definitions in 64 bits ------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("logprobs", "policy"):
        V, t = case["vocab"], s["targets"]
        live = t != IGNORE
        M = t.numel()
        logp = torch.zeros(M, device="cuda", dtype=torch.float64)
        lse = torch.zeros_like(logp)
        for a in range(0, M, 512):
            x = s["logits"][a:a + 512, :V].double()
            z = torch.logsumexp(x, 1)
            lse[a:a + 512] = z * live[a:a + 512]
            pick = torch.arange(x.shape[0], device="cuda"), t[a:a + 512].clamp_min(0)
            logp[a:a + 512] = (x[pick] - z) * live[a:a + 512]
        if op == "logprobs":
            out, coef = {"logp": logp, "lse": lse}, live.double()
            if not case["grad"]:
                return out
        else:
            # derivatives by hand: d/dlogp of -min(r A, clip(r) A) is -r A where the first is the smaller (or both are
            # equal), else 0; of e^d - d - 1 with d = ref - logp it is 1 - e^d
            w = live / live.sum().clamp_min(1).double() if s["weights"] is None else s["weights"].double() * live
            A = s["adv"].double()
            r = torch.exp((logp - s["old"].double()) * live)
            c = torch.minimum(torch.maximum(r, torch.full_like(r, 1 - CLIP_LOW)), torch.full_like(r, 1 + CLIP_HIGH))
            free = r * A <= c * A
            per, coef = torch.where(free, -r * A, -c * A), torch.where(free, -r * A, torch.zeros_like(r))
            k = torch.zeros_like(r)
            if s["ref"] is not None:
                d = (s["ref"].double() - logp) * live
                k = torch.exp(d) - d - 1
                per, coef = per + KL_COEF * k, coef + KL_COEF * (1 - torch.exp(d))
            coef = coef * w
            out = {"loss": (w * per).sum(), "stats": torch.stack([(w * k).sum(), (w * (~free).double()).sum()]), "logp": logp}
        grad = torch.zeros(s["logits"].shape, device="cuda", dtype=torch.float64)
        for a in range(0, M, 512):
            b = min(M, a + 512)
            p = torch.softmax(s["logits"][a:b, :V].double(), 1)
            p[torch.arange(b - a, device="cuda"), t[a:b].clamp_min(0)] -= 1
            grad[a:b, :V] = -coef[a:b, None] * p
        out["grad"] = grad
        return out
    if op == "preference":
        P, live = case["pairs"], (s["targets"] != IGNORE).double()
        ref = 0.0 if s["ref"] is None else s["ref"].double()
        tot = ((s["logp"].double() - ref) * live).sum(1)
        z = BETA * (tot[:P] - tot[P:])
        loss = -((1 - SMOOTHING) * torch.nn.functional.logsigmoid(z) + SMOOTHING * torch.nn.functional.logsigmoid(-z)).sum() / P
        dz = (-(1 - SMOOTHING) * torch.sigmoid(-z) + SMOOTHING * torch.sigmoid(z)) / P
        return {"loss": loss, "rewards": BETA * tot.view(2, P), "dlogp": live * torch.cat([BETA * dz, -BETA * dz])[:, None]}
    # 8-bit format, apart from the plain form: the least exponent by comparison, codes by half-even rounding
    def codes(x):
        M, N = x.shape
        out = torch.empty_like(x)
        for a in range(0, N, BLOCK):
            xb = x[:, a:a + BLOCK]
            top = xb.abs().amax(1, keepdim=True)
            e = torch.ceil(torch.log2((top / 127).clamp_min(2.0 ** -126)))
            e = torch.where(127 * torch.exp2(e - 1) >= top, e - 1, e)
            e = torch.where(127 * torch.exp2(e) < top, e + 1, e).clamp_min(-126)
            out[:, a:a + BLOCK] = torch.round(xb / torch.exp2(e)) * torch.exp2(e)
        return out

    if op == "act8":
        x = codes(s["x"].double())
        if not case["gelu"]:
            return {"x": x}
        return {"x": x, "gelu": torch.nn.functional.gelu(x, approximate="tanh")}
    w, b = s["w"].double(), s["b"].double()
    if not case["back"]:
        x = s["x"].double()
        var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
        xh = (x - mean) / torch.sqrt(var + EPS)
        return {"y": xh * w + b, "kept": codes(xh), "rstd": (var[:, 0] + EPS) ** -0.5}
    N = case["cols"]
    block = torch.arange(N, device="cuda") // BLOCK
    xh = s["q"].double() * torch.exp2(s["e"].double() - 127)[:, block]
    dy, r = s["dy"].double(), s["rstd"].double()[:, None]
    a = dy * w
    new = s["dres_in"].double() + r * (a - a.sum(1, keepdim=True) / N - xh * (a * xh).sum(1, keepdim=True) / N)
    return {"dres": new, "dres16": new, "y": xh * w + b, "dgamma": (dy * xh).sum(0), "dbeta": dy.sum(0)}
