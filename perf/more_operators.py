"""Decoding from a paged key/value cache: plain forms, kernels, and the cases they are timed on.

Operators (``case["op"]``):

* ``store``   K and V of new tokens written into the pages of a cache (16 bits, or quantised to 8), and read back
* ``attend``  attention of one new token per sequence over its pages
* ``sample``  a token per row of logits, by temperature, top-k, top-p and min-p, from given uniform numbers

A cache is ``k_pages`` and ``v_pages`` [pages, heads, page size, head dim]; in 8 bits it holds signed codes, and
``k_exp`` and ``v_exp`` [pages, heads, page size] the exponent byte of each head of each token. Token t of a sequence is
slot ``table[sequence, t // page size] * page size + t % page size``.

``run`` computes the plain form (elementary torch operations) while ``own`` is false and calls the framework's kernels
(``heiretsu_b200.ops.kernels``) while it is true.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HEADS = [(12, 12, 64), (25, 25, 64), (20, 20, 64), (32, 8, 128), (8, 1, 128), (16, 2, 64), (20, 4, 64), (8, 8, 32), (8, 8, 16)]


def listed():
    return [
        # one decoding step of 16 sequences at GPT-2 small's heads: the new K and V, quantised (latency)
        {"name": "store step 16", "op": "store", "tokens": 16, "heads": 12, "kv_heads": 12, "dim": 64, "page": 64, "type": "bf16", "bits": 8},
        # prompts of 8 x 1024 tokens at GPT-2 large's heads, quantised
        {"name": "store prompts 8k 8-bit", "op": "store", "tokens": 8192, "heads": 20, "kv_heads": 20, "dim": 64, "page": 64, "type": "bf16", "bits": 8},
        # an odd number of prompt tokens, fp16 kept as it is, small pages
        {"name": "store prompts 4099 fp16", "op": "store", "tokens": 4099, "heads": 12, "kv_heads": 12, "dim": 64, "page": 16, "type": "fp16", "bits": 16},
        # a single short conversation, GPT-2 small's heads (latency)
        {"name": "attend 1x57", "op": "attend", "seqs": 1, "most": 57, "heads": 12, "kv_heads": 12, "dim": 64, "page": 64, "type": "bf16", "bits": 16},
        # 61 sampled answers of up to GPT-2's 1024 positions
        {"name": "attend 61x1024", "op": "attend", "seqs": 61, "most": 1024, "heads": 12, "kv_heads": 12, "dim": 64, "page": 64, "type": "bf16", "bits": 16},
        # 256 sampled answers at GPT-2 large's heads from the 8-bit cache
        {"name": "attend 256x1024 8-bit", "op": "attend", "seqs": 256, "most": 1024, "heads": 20, "kv_heads": 20, "dim": 64, "page": 64, "type": "bf16", "bits": 8},
        # one long document, 4 query heads to a K/V head, fp16: the work is the split over the length
        {"name": "attend 1x100003 fp16", "op": "attend", "seqs": 1, "most": 100003, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "type": "fp16", "bits": 16},
        # a full server: 64 conversations of up to 8192 tokens, 4 query heads to a K/V head
        {"name": "attend 64x8192", "op": "attend", "seqs": 64, "most": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "type": "bf16", "bits": 16},
        # one sequence with sample.py's settings (latency)
        {"name": "sample 1", "op": "sample", "rows": 1, "vocab": 50257, "type": "bf16", "pad": True, "temperature": 0.8, "top_k": 200, "top_p": 1.0, "min_p": 0.0, "mixed": False},
        # 64 answers to be scored: the model's own distribution, nothing cut off, 32-bit logits
        {"name": "sample 64 whole fp32", "op": "sample", "rows": 64, "vocab": 50257, "type": "fp32", "pad": False, "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "mixed": False},
        # 256 answers, nucleus
        {"name": "sample 256 nucleus", "op": "sample", "rows": 256, "vocab": 50257, "type": "bf16", "pad": True, "temperature": 0.9, "top_k": 0, "top_p": 0.9, "min_p": 0.0, "mixed": False},
        # a server's batch: every row has settings of its own, some take the most likely token
        {"name": "sample 101 mixed", "op": "sample", "rows": 101, "vocab": 32003, "type": "fp16", "pad": False, "temperature": 1.0, "top_k": 50, "top_p": 0.95, "min_p": 0.02, "mixed": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "attend", "attend", "sample"])
    if op == "store":
        heads, kv, dim = rng.choice(HEADS)
        return {"op": op, "tokens": _log(rng, 1, 8192 * 1280 // (kv * dim)), "heads": heads, "kv_heads": kv, "dim": dim,
                "page": rng.choice([16, 32, 64, 128, 48]), "type": rng.choice(["bf16", "fp16"]), "bits": rng.choice([8, 16])}
    if op == "attend":
        heads, kv, dim = rng.choice(HEADS)
        most = _log(rng, 1, 131072)
        seqs = _log(rng, 1, max(1, min(256, 64 * 8192 * 1024 // (most * kv * dim))))
        return {"op": op, "seqs": seqs, "most": most, "heads": heads, "kv_heads": kv, "dim": dim,
                "page": rng.choice([16, 32, 64, 128, 48]), "type": rng.choice(["bf16", "fp16"]), "bits": rng.choice([8, 16])}
    vocab = _log(rng, 1000, 130000)
    return {"op": op, "rows": _log(rng, 1, min(512, 256 * 50257 // vocab)), "vocab": vocab, "type": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
            "pad": rng.random() < 0.5, "temperature": round(rng.uniform(0.3, 1.5), 2), "top_k": rng.choice([0, 0, 1, _log(rng, 2, 1000)]),
            "top_p": rng.choice([1.0, round(rng.uniform(0.05, 0.99), 2)]), "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.3), 3)]),
            "mixed": rng.random() < 0.3}


# ---- inputs ----------------------------------------------------------------------
def _lengths(case):
    """Cached tokens of each sequence: the longest, and others spread over the whole range. The same for every seed, so that
    the work is; the seed deals them out."""
    rng = random.Random(case["seqs"] * 1000003 + case["most"])
    return [case["most"]] + [rng.randint(1, case["most"]) for _ in range(case["seqs"] - 1)]


def _kv(shape, g):
    """Keys and values as a trained model has them: unlike channels, a few of them with an offset."""
    *_, heads, dim = shape
    size = 0.5 + torch.rand(heads, dim, device="cuda", generator=g)
    offset = 3.0 * torch.randn(heads, dim, device="cuda", generator=g) * (torch.rand(heads, dim, device="cuda", generator=g) < 0.05)
    return torch.randn(shape, device="cuda", generator=g).mul_(size).add_(offset)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dt, s = case["op"], TYPES[case["type"]], {"case": case}
    if op == "sample":
        M, V = case["rows"], case["vocab"]
        W = (V + 127) // 128 * 128 if case["pad"] else V
        # logits of a trained model: normal, with a few hundred plausible tokens raised by up to 14
        x = torch.randn(M, V, device="cuda", generator=g).mul_(2.0)
        likely = torch.randint(0, V, (M, 200), device="cuda", generator=g)
        x.scatter_add_(1, likely, 14 * torch.rand(M, 1, device="cuda", generator=g) * torch.rand(M, 200, device="cuda", generator=g).square())
        s["logits"] = torch.zeros(M, W, device="cuda", dtype=dt)
        s["logits"][:, :V] = x
        s["u"] = torch.rand(M, device="cuda", generator=g)
        if case["mixed"]:
            r = torch.rand(4, M, device="cuda", generator=g)
            s["temperature"] = torch.where(r[0] < 0.2, 0.0, 0.5 + case["temperature"] * r[0])
            s["top_k"] = torch.where(r[1] < 0.3, 0, 1 + (2 * case["top_k"] * r[1]).long())
            s["top_p"] = torch.where(r[2] < 0.3, 1.0, case["top_p"] * r[2])
            s["min_p"] = torch.where(r[3] < 0.5, 0.0, case["min_p"] * r[3])
        else:
            s |= {k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")}
        return s
    H, D, ps = case["kv_heads"], case["dim"], case["page"]
    if op == "store":
        N = case["tokens"]
        pages = (N + ps - 1) // ps + 3
        s["qkv"] = _kv((N, case["heads"] + 2 * H, D), g).to(dt).view(N, -1)  # what the projection leaves: [Q | K | V] of each token
        # whole pages in any order, as an allocator deals them out
        order = torch.randperm(pages, device="cuda", generator=g)
        s["slots"] = (order[:, None] * ps + torch.arange(ps, device="cuda")).view(-1)[:N].contiguous()
        kind = torch.int8 if case["bits"] == 8 else dt
        s["pools"] = {n: torch.zeros(pages, H, ps, D, device="cuda", dtype=kind) for n in ("k_pages", "v_pages")}
        if case["bits"] == 8:
            s["pools"] |= {n: torch.zeros(pages, H, ps, device="cuda", dtype=torch.uint8) for n in ("k_exp", "v_exp")}
        return s
    B = case["seqs"]
    lengths = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)[torch.randperm(B, device="cuda", generator=g)]
    need = (lengths + ps - 1) // ps
    wide = (case["most"] + ps - 1) // ps
    pages = sum((n + ps - 1) // ps for n in _lengths(case))
    order = torch.randperm(pages, device="cuda", generator=g).int()
    live = torch.arange(wide, device="cuda")[None] < need[:, None]
    s["table"] = torch.full((B, wide), -1, device="cuda", dtype=torch.int32)
    s["table"][live] = order
    s["lengths"] = lengths
    s["q"] = (2 * torch.randn(B, case["heads"] * D, device="cuda", generator=g)).to(dt)
    s["pools"] = {}
    for n in ("k", "v"):
        x = _kv((pages, ps, H, D), g).transpose(1, 2).to(dt)
        if case["bits"] == 8:
            codes, e = _quantise(x)
            s["pools"][n + "_exp"] = e
            x = codes
        s["pools"][n + "_pages"] = x.contiguous()
    return s


def _new(s):
    """K and V [tokens, heads, dim] of a projection's output: views of it."""
    case = s["case"]
    return s["qkv"].view(case["tokens"], -1, case["dim"]).split([case["heads"], case["kv_heads"], case["kv_heads"]], 1)[1:]


# ---- plain forms -----------------------------------------------------------------
def _quantise(x):
    """x [..., D] -> (codes int8 [..., D], exponent bytes [...]): 2^e is the least power of two, e >= -126, with
    max|x| <= 127 * 2^e; the byte is e + 127, a code is x / 2^e rounded to the nearest whole number, ties to even."""
    mant, ex = torch.frexp(x.abs().amax(-1).float())  # max|x| = mant * 2^ex, mant in [0.5, 1)
    e = torch.where(mant * 128 > 127, ex - 6, ex - 7).clamp_min_(-126)
    e = torch.where(mant == 0, torch.full_like(e, -126), e)
    return torch.ldexp(x.float(), -e[..., None].float()).round_().to(torch.int8), (e + 127).to(torch.uint8)


def _values(codes, exps):
    return codes.float() * torch.ldexp(torch.ones((), device=codes.device), exps.float() - 127)[..., None]


def _store(s):
    case, pools = s["case"], s["pools"]
    H, D, ps = case["kv_heads"], case["dim"], case["page"]
    page, at = s["slots"] // ps, s["slots"] % ps
    out = {}
    k, v = _new(s)
    k_pages, v_pages = pools["k_pages"], pools["v_pages"]
    if case["bits"] == 8:
        k_exp, v_exp = pools["k_exp"], pools["v_exp"]
        k_pages[page, :, at], k_exp[page, :, at] = _quantise(k)
        v_pages[page, :, at], v_exp[page, :, at] = _quantise(v)
        out["k"] = _values(k_pages[page, :, at], k_exp[page, :, at]).to(k.dtype)
        out["v"] = _values(v_pages[page, :, at], v_exp[page, :, at]).to(v.dtype)
        return out
    k_pages[page, :, at], v_pages[page, :, at] = k, v
    return {"k": k_pages[page, :, at], "v": v_pages[page, :, at]}


def _gathered(pools, name, table, ps):
    """[B, heads, tokens, D] in 32 bits of the pages in the table's rows."""
    pages = table.clamp_min(0).long()
    x = pools[name + "_pages"][pages]  # [B, pages, heads, ps, D]
    x = _values(x, pools[name + "_exp"][pages]) if name + "_exp" in pools else x.float()
    B, n, H, _, D = x.shape
    return x.transpose(1, 2).reshape(B, H, n * ps, D)


def _attend(s):
    case = s["case"]
    B, D, G = case["seqs"], case["dim"], case["heads"] // case["kv_heads"]
    q = s["q"].float().view(B, -1, G, D)
    x = _gathered(s["pools"], "k", s["table"], case["page"])
    x = q @ x.transpose(2, 3) / math.sqrt(D)
    dead = torch.arange(x.shape[-1], device="cuda") >= s["lengths"][:, None, None, None]
    x.masked_fill_(dead, -math.inf)
    top = x.amax(-1, keepdim=True)
    w = (x - top).exp_()
    total = w.sum(-1, keepdim=True)
    out = (w @ _gathered(s["pools"], "v", s["table"], case["page"])) / total
    return {"out": out.to(s["q"].dtype).view(B, -1, D), "lse": (top + total.log()).view(B, -1)}


def _sample(s):
    """In 64 bits: which token a number falls on is a comparison of sums."""
    case = s["case"]
    M, V = case["rows"], case["vocab"]
    per_row = lambda v: torch.as_tensor(v, device="cuda", dtype=torch.float64).expand(M)[:, None]  # noqa: E731
    t, k, p, least = (per_row(s[n]) for n in ("temperature", "top_k", "top_p", "min_p"))
    x = s["logits"][:, :V].double()
    x, order = x.sort(dim=1, descending=True, stable=True)  # equal logits: lowest index first
    x = (x - x[:, :1]) / torch.where(t > 0, t, 1.0)
    rank = torch.arange(V, device="cuda")[None]
    w = torch.where((rank < k) | (k < 1), x.exp(), 0.0)
    before = w.cumsum(1) - w
    kept = (before < p * w.sum(1, keepdim=True)) & (x >= least.log())
    kept = torch.where(t > 0, kept, False) | (rank == 0)
    w = torch.zeros_like(w).scatter_(1, order, torch.where(kept, w, 0.0))  # back in the vocabulary's order
    reached = w.cumsum(1)
    return {"tokens": (reached > s["u"].double()[:, None] * reached[:, -1:]).int().argmax(1)}


# ---- the framework's calls ---------------------------------------------------------
def _calls(s):
    from heiretsu_b200.ops import kernels as K

    case = s["case"]
    if case["op"] == "store":
        k, v = _new(s)
        K.kv_write(k, v, s["slots"], **s["pools"])
        k, v = K.kv_read(s["slots"], **s["pools"], dtype=k.dtype)
        return {"k": k, "v": v}
    if case["op"] == "attend":
        q = s["q"].view(case["seqs"], case["heads"], case["dim"])
        out, lse = K.decode_attention(q, table=s["table"], lengths=s["lengths"], **s["pools"])
        return {"out": out, "lse": lse}
    return {"tokens": K.sample_tokens(s["logits"], case["vocab"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                      top_p=s["top_p"], min_p=s["min_p"])}


def run(state):
    if own:
        return _calls(state)
    return {"store": _store, "attend": _attend, "sample": _sample}[state["case"]["op"]](state)


def work(case):
    """Bytes: every input read once and every output written once. Flops: one per elementary step of the formula."""
    if case["op"] == "sample":
        M, V, es = case["rows"], case["vocab"], 4 if case["type"] == "fp32" else 2
        return {"bytes": M * (V * es + 4 + 8 + (20 if case["mixed"] else 0)), "flops": M * V * 5}
    token = 2 * case["kv_heads"] * (2 * case["dim"] if case["bits"] == 16 else case["dim"] + 1)  # K and V of a cached token
    if case["op"] == "store":  # written in one call, read in another: what is kept crosses memory twice
        n = case["tokens"]
        return {"bytes": n * (2 * 4 * case["kv_heads"] * case["dim"] + 2 * token + 16), "flops": n * case["kv_heads"] * case["dim"] * 4}
    n, B = sum(_lengths(case)), case["seqs"]
    pages = sum((x + case["page"] - 1) // case["page"] for x in _lengths(case))
    return {"bytes": n * token + B * (case["heads"] * (4 * case["dim"] + 4) + 4) + 4 * pages, "flops": 4 * n * case["heads"] * case["dim"]}


# ---- the definitions in 64 bits ------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store":
        k, v = _new(s)
        if case["bits"] == 16:
            return {"k": k.double(), "v": v.double()}

        def kept(x):  # the least exponent by comparison
            x = x.double()
            top = x.abs().amax(-1, keepdim=True)
            e = torch.ceil(torch.log2((top / 127).clamp_min(2.0 ** -126)))
            e = torch.where(127 * torch.exp2(e - 1) >= top, e - 1, e)
            e = torch.where(127 * torch.exp2(e) < top, e + 1, e).clamp_min(-126)
            return torch.round(x / torch.exp2(e)) * torch.exp2(e)

        return {"k": kept(k), "v": kept(v)}
    if case["op"] == "attend":
        # a sequence and K/V head at a time, over the tokens it has and no others
        D, ps, G = case["dim"], case["page"], case["heads"] // case["kv_heads"]
        q = s["q"].double().view(case["seqs"], case["kv_heads"], G, D)
        out, lse = torch.empty_like(q), torch.empty(q.shape[:3], device="cuda", dtype=torch.float64)
        for b, n in enumerate(s["lengths"].tolist()):
            at = torch.arange(n, device="cuda")
            page = s["table"][b].long()[at // ps]
            k, v = (s["pools"][m][page, :, at % ps].double().transpose(0, 1) for m in ("k_pages", "v_pages"))
            if case["bits"] == 8:
                k, v = (x * torch.exp2(s["pools"][m][page, :, at % ps].double() - 127).t()[..., None] for x, m in ((k, "k_exp"), (v, "v_exp")))
            x = torch.einsum("hgd,htd->hgt", q[b], k) * D ** -0.5
            lse[b] = torch.logsumexp(x, -1)
            out[b] = torch.einsum("hgt,htd->hgd", torch.exp(x - lse[b][..., None]), v)
        return {"out": out.reshape(case["seqs"], -1, D), "lse": lse.reshape(case["seqs"], -1)}
    # a row at a time, over its different logits: how many have each, and where the last one kept is
    tokens = []
    setting = lambda n, i: float(s[n][i]) if torch.is_tensor(s[n]) else float(s[n])  # noqa: E731
    for i in range(case["rows"]):
        x = s["logits"][i, : case["vocab"]].double().cpu()
        if setting("temperature", i) <= 0:
            tokens.append(int((x == x.max()).nonzero()[0]))
            continue
        level, count = torch.unique(x, return_counts=True)
        level, count = level.flip(0), count.flip(0)
        k = int(setting("top_k", i))
        if k > 0:
            count = torch.minimum(count, (k - (count.cumsum(0) - count)).clamp_min(0))
        m = torch.exp((level - level[0]) / setting("temperature", i))
        reach = setting("top_p", i) * (m * count).sum()
        ahead = (m * count).cumsum(0) - m * count
        # of `count` equal ones the j-th is kept if ahead + j m < reach
        fit = torch.ceil((reach - ahead) / m.clamp_min(1e-300)).clamp_min(0)
        count = torch.minimum(count.double(), fit)
        count[m < setting("min_p", i)] = 0
        count[0] = count[0].clamp_min(1)
        last = int((count > 0).nonzero()[-1])
        mass = torch.where(x >= level[last], torch.exp((x - level[0]) / setting("temperature", i)), 0.0)
        ties = (x == level[last]).nonzero()[:, 0]
        mass[ties[int(count[last]):]] = 0
        reached = mass.cumsum(0)
        tokens.append(int((reached > float(s["u"][i]) * reached[-1]).nonzero()[0]))
    return {"tokens": torch.tensor(tokens, device="cuda")}
