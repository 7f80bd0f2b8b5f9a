"""Post-training objectives and 8-bit activations without a GPU: the plain PyTorch path against 64-bit oracles and
finite differences, and the fused path's host code with its kernels replaced by stand-ins (post_emulation.py)."""
import pytest
import torch

import post_emulation
import post_oracle as O
from heiretsu_b200.config import GPTConfig
from heiretsu_b200.models.gpt import GPT

CFG = dict(block_size=64, vocab_size=200, n_layer=2, n_head=2, n_embed=128)
IGNORE = -100


def batch(n=4, T=48, seed=5):
    g = torch.Generator().manual_seed(seed)
    idx = torch.randint(0, 200, (n, T), generator=g)
    tgt = torch.randint(0, 200, (n, T), generator=g)
    tgt[torch.rand(n, T, generator=g) < 0.3] = IGNORE
    old = -5.3 + 0.3 * torch.randn(n, T, generator=g)
    ref = -5.3 + 0.3 * torch.randn(n, T, generator=g)
    adv = torch.randn(n, T, generator=g)
    return idx, tgt, old, ref, adv


def plain(dtype=torch.float64, moe=False):
    torch.manual_seed(0)
    kw = dict(num_experts=2, top_k=1, moe_freq=2) if moe else {}
    return GPT(GPTConfig(**CFG, dropout=0.0, **kw)).to(dtype)


def fused(recompute=False, act_bits=16, dropout=0.0):
    from heiretsu_b200.parallel.flat import FlatParams

    torch.manual_seed(0)
    m = GPT(GPTConfig(**CFG, dropout=dropout))
    flat = FlatParams(m, torch.device("cpu"))
    m.fused, m.recompute, m.act_bits = True, recompute, act_bits
    if dropout > 0:
        seed = torch.tensor([77], dtype=torch.int32)
        for layer, blk in enumerate(m.tr.h):
            blk._hb_dropout = (seed, layer, dropout)
    return m, flat


def run(m, kind, b, **kw):
    """(loss, what else the objective returns) of one objective."""
    idx, tgt, old, ref, adv = b
    if kind == "logp":  # any loss of the log-probabilities
        lp = m.token_logprobs(idx, tgt)
        return (lp * adv.to(lp.dtype)).sum() / 50, (lp.detach(),)
    if kind == "policy":
        loss, aux, stats, lp = m.policy_loss(idx, tgt, old, adv, ref_logp=ref, clip_high=0.25, kl_coef=0.1, **kw)
        return loss + aux, (stats, lp)
    loss, aux, rewards = m.preference_loss(idx, tgt, ref_logp=ref, beta=0.3, label_smoothing=0.1, **kw)
    return loss + aux, (rewards,)


def oracle(m, kind, b):
    idx, tgt, old, ref, adv = b
    with torch.no_grad():
        logits = m(idx)[0]
    lp, _, _ = O.logprobs(logits.reshape(-1, 200), 200, tgt.reshape(-1))
    live = tgt.reshape(-1) != IGNORE
    if kind == "logp":
        return (lp * adv.reshape(-1)).sum() / 50, (lp.view(idx.shape),)
    if kind == "policy":
        loss, stats, _ = O.policy(lp, live, old.reshape(-1), adv.reshape(-1), ref.reshape(-1), None, 0.2, 0.25, 0.1)
        return loss, (stats, lp.view(idx.shape))
    loss, rewards, _ = O.preference(lp.view(idx.shape), tgt, ref, 0.3, 0.1)
    return loss, (rewards,)


KINDS = ["logp", "policy", "preference"]


@pytest.mark.parametrize("kind", KINDS)
def test_plain_values(kind):
    m, b = plain(), batch()
    loss, rest = run(m, kind, b)
    want, wrest = oracle(m, kind, b)
    # the plain path takes log-probabilities in 32 bits: 2^-24 of values around 5, a few roundings each; sums of 100
    assert abs(loss.item() - want.item()) <= 1e-5 * (1 + abs(want.item()))
    for a, c in zip(rest, wrest):
        assert torch.allclose(a.double(), c.double(), atol=3e-5, rtol=1e-5)
    counts = b[1] != IGNORE
    if kind != "preference":
        assert (rest[-1][~counts] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
def test_plain_gradients_against_differences(kind):
    """Central differences along random parameter directions in a 64-bit model: the loss's 32-bit log-probabilities
    leave about 1e-6 / h, curvature h^2."""
    m, b = plain(), batch()
    loss, _ = run(m, kind, b)
    params = [p for p in m.parameters() if p.requires_grad]
    grads = torch.autograd.grad(loss, params)
    g = torch.Generator().manual_seed(1)
    h = 2e-2
    for _ in range(3):
        v = [torch.randn(p.shape, generator=g, dtype=p.dtype) for p in params]
        norm = sum(x.square().sum() for x in v).sqrt()
        vals = []
        for s in (h, -h):
            with torch.no_grad():
                for p, x in zip(params, v):
                    p.add_(s / norm * x)
                vals.append(oracle(m, kind, b)[0].item())
                for p, x in zip(params, v):
                    p.sub_(s / norm * x)
        num = (vals[0] - vals[1]) / (2 * h)
        ana = sum((gr * x).sum() for gr, x in zip(grads, v)).item() / norm.item()
        assert abs(num - ana) <= 1e-4 + 2 * h * h, (num, ana)


def test_plain_with_moe_and_sequence_advantages():
    m, b = plain(torch.float32, moe=True), batch()
    loss, aux, _, _ = m.policy_loss(b[0], b[1], b[2], b[4][:, 0])
    same, _, _, _ = m.policy_loss(b[0], b[1], b[2], b[4][:, :1].expand(4, 48))
    assert torch.equal(loss, same) and aux > 0
    (loss + aux).backward()
    w = torch.rand(4, 48)
    a, _, _, _ = m.policy_loss(b[0], b[1], b[2], b[4], weights=w)
    n, _, _, _ = m.policy_loss(b[0], b[1], b[2], b[4], weights=2 * w)
    assert abs(n.item() - 2 * a.item()) <= 1e-5 * (1 + abs(a.item()))


def test_nothing_counts():
    m, b = plain(torch.float32), batch()
    none = torch.full_like(b[1], IGNORE)
    loss, _, stats, lp = m.policy_loss(b[0], none, b[2], b[4], ref_logp=b[3])
    assert loss.item() == 0 and (stats == 0).all() and (lp == 0).all()
    loss.backward()
    loss, _, rewards = m.preference_loss(b[0], none, ref_logp=b[3])
    assert abs(loss.item() - 0.6931472) < 1e-6 and (rewards == 0).all()


def test_targets_that_are_no_tokens_give_nan():
    m, b = plain(torch.float32), batch()
    tgt = b[1].clone()
    tgt[0, 40], tgt[1, 41], tgt[2, 42] = 200, -1, IGNORE
    lp = m.token_logprobs(b[0], tgt)
    assert torch.isnan(lp[0, 40]) and torch.isnan(lp[1, 41]) and lp[2, 42] == 0
    assert torch.isnan(lp).sum() == 2


def test_refusals():
    m, b = plain(torch.float32), batch(3)
    idx, tgt, old, ref, adv = b
    for call in (lambda: m.preference_loss(idx, tgt), lambda: m.token_logprobs(idx, tgt[:, :5]),
                 lambda: m.policy_loss(idx, tgt, old[:, :4], adv), lambda: m.policy_loss(idx, tgt, old, adv[:2]),
                 lambda: m.policy_loss(idx, tgt, old, adv, ref_logp=ref.reshape(-1)),
                 lambda: m.token_logprobs(idx.repeat(1, 3), tgt.repeat(1, 3))):
        with pytest.raises(ValueError):
            call()


def grads(m, loss):
    loss.backward()
    return {n: p.main_grad.clone() for n, p in m.named_parameters()}


def close(a, b, tol):
    for n in a:
        assert (a[n] - b[n]).norm().item() <= tol * (b[n].norm().item() + 1e-8), (n, ((a[n] - b[n]).norm() / b[n].norm()).item())


@pytest.mark.parametrize("upstream", [1.0, 0.25])
@pytest.mark.parametrize("kind", KINDS)
def test_fused_host_code(monkeypatch, kind, upstream):
    """Loss and every gradient of the fused path (16-bit emulated kernels) against the plain model."""
    post_emulation.emulate(monkeypatch)
    b = batch()
    m, flat = fused()
    loss, rest = run(m, kind, b)
    p = plain(torch.float32)
    want, wrest = run(p, kind, b)
    assert abs(loss.item() - want.item()) < 2e-2
    (upstream * want).backward()
    close(grads(m, upstream * loss), {n: q.grad for n, q in p.named_parameters()}, 5e-2)


def test_fused_scoring_keeps_nothing(monkeypatch):
    post_emulation.emulate(monkeypatch)
    b = batch()
    m, flat = fused()
    with torch.no_grad():
        lp = m.token_logprobs(b[0], b[1])
        loss, aux, rewards = m.preference_loss(b[0], b[1], ref_logp=lp)
    assert not lp.requires_grad and abs(loss.item() - 0.6931472) < 1e-6 and (rewards == 0).all()
    loss, _, stats, _ = m.policy_loss(b[0], b[1], lp, b[4], ref_logp=lp, kl_coef=1.0)
    # the model against itself: ratios of 1 but for the scores' rounding, (2^-24 * 5)^2 / 2
    assert stats[0] <= 1e-12 and stats[1] == 0


# An 8-bit code is off by at most half a step, the step is at most 2 max / 127, and 128 normal values reach about 2.7
# standard deviations: at most 1.2% of the standard deviation (root mean square) per kept value. A parameter's gradient
# is linear in at most 4 such values a layer, over 2 layers; errors of unlike origin add in squares to
# 1.2% sqrt(8) = 3.5%, and the softmax's derivative at most doubles an error of its scores (|p - 1| <= 1, twice).
ACT8_TOL = 0.07


@pytest.mark.parametrize("dropout", [0.0, 0.2])
@pytest.mark.parametrize("recompute", [False, True])
def test_act8_gradients(monkeypatch, recompute, dropout):
    post_emulation.emulate(monkeypatch)
    b = batch()
    m16, f16 = fused(dropout=dropout)
    m8, f8 = fused(recompute=recompute, act_bits=8, dropout=dropout)
    l16, _ = run(m16, "policy", b)
    l8, _ = run(m8, "policy", b)
    assert abs(l8.item() - l16.item()) < 1e-6  # the forward is the same
    close(grads(m8, l8), grads(m16, l16), ACT8_TOL)


def test_act8_keeps_fewer_bytes(monkeypatch):
    """A dense block keeps (1 + 3 + 1 + 1 + 4) H code bytes a token, one exponent per 128, and the softmax statistics
    and two rstd, against 36 H."""
    import heiretsu_b200.models.fused as FZ

    post_emulation.emulate(monkeypatch)

    def size(o):
        if torch.is_tensor(o):
            return o.numel() * o.element_size()
        if isinstance(o, FZ._Act8):
            return size(o.norm) + size(o.rest)
        if isinstance(o, FZ._Recompute):
            return size(o.x_in)
        return sum(size(x) for x in o) if isinstance(o, (tuple, list)) else 0

    held = {}
    for key, bits, rec in (("16", 16, False), ("8", 8, False), ("in16", 16, True), ("in8", 8, True)):
        m, flat = fused(recompute=rec, act_bits=bits)
        kept = []
        real = FZ._Body.apply
        loss, _ = run(m, "logp", batch())
        node = loss.grad_fn
        seen, todo = set(), [node]
        while todo:
            n = todo.pop()
            if n is None or n in seen:
                continue
            seen.add(n)
            if type(n).__name__ == "_BodyBackward":
                kept = n.saved
            todo += [f for f, _ in n.next_functions]
        held[key] = size(kept) / (2 * 4 * 48 * 128)  # per layer, token and channel
    lse = 2 * 64 * 4 * 2 / 48 / 128  # [heads, T padded to 128] fp32 over 48 tokens and 128 channels
    assert held["16"] >= 36 and held["8"] <= 10 + 10 / 128 + 8 / 128 + 2 * lse, held
    assert held["in16"] == 4 and held["in8"] <= 1 + 1 / 128


def test_act8_bits_are_checked(monkeypatch):
    from heiretsu_b200.models.fused import blocks_fused

    post_emulation.emulate(monkeypatch)
    m, flat = fused(act_bits=4)
    with pytest.raises(ValueError, match="16 or 8"):
        run(m, "logp", batch())


def test_trainer_refuses_8_bits_on_the_plain_engine():
    from heiretsu_b200.topo import Topology
    from heiretsu_b200.trainer import Engine, build_argparser

    args = build_argparser().parse_args(["--activation_bits", "8", "--n_layer", "1", "--n_head", "2", "--n_embed", "128"])
    topo = Topology(dp=1, ep=1, tp=1, pp=1, rank=0, world_size=1, dp_rank=0, ep_rank=0, pp_rank=0, tp_rank=0,
                    tp_group=None, pp_group=None, ep_group=None, dp_group=None)
    with pytest.raises(ValueError, match="activation_bits"):
        Engine(args, topo, torch.device("cpu"), GPTConfig(**CFG))


def test_cpu_tensors_are_refused_by_the_kernels():
    from heiretsu_b200.ops import kernels as K
    from heiretsu_b200.ops._C import available

    if not available():
        pytest.skip("extension not built")
    x, t, f = torch.zeros(4, 128), torch.zeros(4, dtype=torch.long), torch.zeros(4)
    q, e = torch.zeros(4, 128, dtype=torch.int8), torch.zeros(4, 1, dtype=torch.uint8)
    w = torch.ones(128)
    for call in (lambda: K.token_logprobs(x, 128, t), lambda: K.policy_loss(x, 128, t, f, f),
                 lambda: K.preference_loss(x, torch.zeros(4, 128, dtype=torch.long)), lambda: K.act8_pack(x),
                 lambda: K.act8_unpack(q, e), lambda: K.act8_unpack_gelu(q, e), lambda: K.layernorm_fwd_act8(x, w, w),
                 lambda: K.layernorm_bwd_act8(x, q, e, f, w, w, x, x, x.bfloat16(), w, w)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_oracle_format():
    """The 8-bit oracle on values whose codes are known."""
    x = torch.zeros(1, 260)
    x[0, 0], x[0, 1], x[0, 2] = 127.0, 0.5, 1.5   # step 1: ties to even
    x[0, 128] = 128.0                             # step 2
    codes, e, bad = O.act8_codes(x)
    assert codes[0, :3].tolist() == [127, 0, 2] and codes[0, 128] == 64
    assert e[0].tolist() == [0, 1, -126] and not bad.any()
    y = O.act8_values(codes, e, bad)
    assert y[0, 128] == 128 and y[0, 2] == 2
