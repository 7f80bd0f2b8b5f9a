"""Post-training objectives where a training program can go wrong: gradients that are infinite at positions that take no
part, values at the ends of a type's range, arguments that are refused. Plain path, and the fused path's host code on
stand-ins."""
import pytest
import torch

import post_emulation
import post_oracle as O
from test_objectives_cpu import IGNORE, batch, fused, grads, plain


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("engine", ["plain", "fused"])
def test_a_derivative_that_is_infinite_at_ignored_tokens(monkeypatch, engine, value):
    """The gradient of ignored tokens' log-probabilities, infinity or NaN, changes no parameter's gradient."""
    post_emulation.emulate(monkeypatch)
    idx, tgt, _, _, adv = batch()
    out = []
    for at_ignored in (0.0, value):
        m = fused()[0] if engine == "fused" else plain(torch.float32)
        lp = m.token_logprobs(idx, tgt)
        lp.backward(torch.where(tgt == IGNORE, torch.full_like(adv, at_ignored), adv))
        out.append({n: (p.main_grad if engine == "fused" else p.grad).clone() for n, p in m.named_parameters()})
    for n in out[0]:
        assert torch.isfinite(out[1][n]).all() and torch.equal(out[0][n], out[1][n]), n


def test_a_loss_of_the_square_root(monkeypatch):
    """sqrt(-logp) over the counted tokens: the fused gradients follow the plain ones (tolerance of the fused host code)."""
    post_emulation.emulate(monkeypatch)
    idx, tgt, _, _, _ = batch()
    m, p = fused()[0], plain(torch.float32)
    loss = [torch.where(tgt != IGNORE, (-q.token_logprobs(idx, tgt)).sqrt(), 0.0).sum() / 100 for q in (m, p)]
    loss[1].backward()
    got = grads(m, loss[0])
    for n, q in p.named_parameters():
        assert (got[n] - q.grad).norm() <= 5e-2 * q.grad.norm() + 1e-8, n


def _spread_head(device, amp, M=64, H=128, V=384):
    """(arguments of the log-probability head, weight): half of the tokens' logits lie about 17 below the others', so that
    their probabilities are 1e-10 to 1e-8."""
    g = torch.Generator().manual_seed(2)
    u = torch.randn(H, generator=g).sign()
    w = 0.05 * torch.randn(V, H, generator=g)
    w[V // 2:] -= 0.19 * u
    w, x = w.to(device), (torch.randn(M, H, generator=g) + u).to(device).requires_grad_(True)
    wte, ln_w, ln_b = (torch.nn.Parameter(t) for t in (w, torch.ones(H, device=device), torch.zeros(H, device=device)))
    for p in (wte, ln_w, ln_b):
        p.main_grad = torch.zeros_like(p)
    wte.w16 = w.to(amp)
    tgt = torch.randint(0, V // 2, (M,), generator=g).to(device)
    tgt[::7] = IGNORE
    return (x, ln_w, ln_b, wte, tgt, V, True), wte


def fp16_range(device, amp):
    """(gradient of the head's weight, that of the formula on the same 16-bit operands, loss scale, probabilities)."""
    from heiretsu_b200.models.objectives import _HeadLogp

    scale = 65536.0
    args, wte = _spread_head(device, amp)
    x, tgt, V = args[0], args[4], args[5]
    logp = _HeadLogp.apply(*args)
    rows = torch.where(tgt != IGNORE, 0.4, 0.0) * scale
    logp.backward(rows)
    xn = torch.nn.functional.layer_norm(x.detach(), x.shape[1:]).to(amp).double()
    p = torch.softmax((xn @ wte.w16.double().t()).to(amp).double(), 1)
    one = torch.nn.functional.one_hot(tgt.clamp_min(0), V)
    return wte.main_grad.double() / scale, ((rows[:, None].double() * (one - p)).t() @ xn) / scale, p


def check_fp16_range(got, want, p):
    """Every token's row, those of probability 1e-9 too. Errors: half a step of the logits (2^-11 of up to 32, or two steps
    where 32-bit sums and the 64-bit one round apart) in p; half a step of the products, 2^-25 absolute where they are
    subnormal: next to 65536 * 0.4 * 1e-9 = 2.6e-5 that is 0.1%."""
    assert torch.isfinite(got).all()
    rare = p.amax(0) < 3e-8
    assert rare.sum() > 20 and (p.amax(0)[rare] > 1e-11).any()
    seen = p.amax(0) > 1e-9
    rel = (got - want).norm(dim=1) / want.norm(dim=1)
    assert (rel[seen] <= 3 * 32 * 2.0 ** -11 + 0.005).all(), rel[seen].max()


def test_fp16_probabilities_keep_their_gradient(monkeypatch):
    """fp16 with a loss scale: dlogp 26214 times hidden states of 3 passes the type's largest value, and
    probabilities below 2^-25 its least one; neither may lose the gradient."""
    post_emulation.emulate(monkeypatch)
    check_fp16_range(*fp16_range("cpu", torch.float16))


@pytest.mark.parametrize("engine", ["plain", "fused"])
def test_balance_loss_beside_the_log_probabilities(monkeypatch, engine):
    """A mixture-of-experts model: the aux loss of ``forward`` and the other objectives, whose gradient reaches the router."""
    idx, tgt, old, _, adv = batch()
    if engine == "plain":
        m = plain(torch.float32, moe=True)
        want = m(idx, tgt.clamp_min(0))[2]
    else:  # dense blocks on the stand-ins: no balance loss, the same form
        post_emulation.emulate(monkeypatch)
        m = fused()[0]
        want = torch.zeros(())
    lp, aux = m.token_logprobs(idx, tgt, return_aux=True)
    assert torch.equal(lp, m.token_logprobs(idx, tgt)) and torch.equal(aux, want)
    assert torch.equal(aux, m.policy_loss(idx, tgt, old, adv)[1])
    if engine == "plain":
        routers = [p for n, p in m.named_parameters() if "router" in n or "gate" in n]
        assert routers and aux > 0
        assert any(g is not None and g.abs().max() > 0 for g in torch.autograd.grad(aux, routers, allow_unused=True))


def overflowing(n=24, device="cpu"):
    """(log-probabilities, old, advantages, reference, weights): ratios and KL terms that 32 bits cannot hold, wherever the
    clip range, an advantage or a weight of 0 takes them out of the loss."""
    logp = torch.linspace(-9, -0.1, n, device=device)
    old, adv, ref, w = logp - 0.05, torch.linspace(-1, 1, n, device=device), logp + 0.1, torch.full((n,), 1 / n, device=device)
    old[3:6], adv[3:6] = -300.0, 0.0                   # no advantage
    old[6:9], adv[6:9] = -300.0, 2.0                   # past the clip range
    old[9:12], adv[9:12], w[9:12] = -300.0, -2.0, 0.0  # no weight
    ref[12:15], w[12:15] = 300.0, 0.0
    return logp, old, adv, ref, w


@pytest.mark.parametrize("kl", [0.0, 0.1])
def test_policy_terms_past_32_bits(kl):
    """Loss, statistics and gradient of the plain form against 64 bits, which hold e^300."""
    from heiretsu_b200.models.objectives import policy_loss_plain

    logp, old, adv, ref, w = (t[None] for t in overflowing())
    if kl == 0:
        ref[0, 15] = 300.0  # counts, in the statistic alone
    lp = logp.clone().requires_grad_(True)
    loss, stats = policy_loss_plain(lp, torch.zeros_like(lp).long(), old, adv, ref, w, 0.2, 0.25, kl)
    loss.backward()
    want, wstats, d = O.policy(logp[0], torch.ones(24, dtype=torch.bool), old[0], adv[0], ref[0], w[0], 0.2, 0.25, kl)
    # 24 terms of at most 2, a few roundings each
    assert abs(loss.item() - want.item()) <= 24 * 2 * 8 * 2.0 ** -24 and stats[1] == wstats[1].float()
    assert (lp.grad[0].double() - d).abs().max() <= 8 * 2.0 ** -24 * d.abs().max()
    if kl:
        assert abs(stats[0].item() - wstats[0].item()) <= 1e-6


@pytest.mark.parametrize("engine", ["plain", "fused"])
def test_only_the_model_is_differentiated(monkeypatch, engine):
    """The first policy step may score its own tokens without no_grad: old log-probabilities, reference, advantages and
    weights are constants on either engine, so the gradients are those of detached ones, not 0."""
    post_emulation.emulate(monkeypatch)
    idx, tgt, _, _, adv = batch()
    out = []
    for constant in (True, False):
        m = fused()[0] if engine == "fused" else plain(torch.float32)
        old = m.token_logprobs(idx, tgt)
        a, w = adv.clone().requires_grad_(True), torch.full_like(adv, 0.01).requires_grad_(True)
        given = [t.detach() if constant else t for t in (old, a, old, w)]
        loss = m.policy_loss(idx, tgt, given[0], given[1], ref_logp=given[2], weights=given[3], kl_coef=0.1)[0]
        loss = loss + m.preference_loss(idx, tgt, ref_logp=given[2])[0]
        loss.backward()
        assert a.grad is None and w.grad is None
        out.append({n: (p.main_grad if engine == "fused" else p.grad).clone() for n, p in m.named_parameters()})
    for n in out[0]:
        assert out[0][n].norm() > 0 and torch.equal(out[0][n], out[1][n]), n


@pytest.mark.parametrize("objective", ["logp", "policy", "preference"])
def test_a_target_that_is_no_token_gives_gradients_of_nan(objective):
    """The plain path as the kernels: a step on such a batch is skipped for its gradient norm, not taken without the token."""
    idx, tgt, old, ref, adv = batch()
    tgt[0, 40] = 200
    m = plain(torch.float32)
    if objective == "logp":
        loss = (m.token_logprobs(idx, tgt) * adv).sum()
    else:
        loss = (m.policy_loss(idx, tgt, old, adv) if objective == "policy" else m.preference_loss(idx, tgt, ref_logp=ref))[0]
    loss.backward()
    assert torch.isnan(loss) and torch.isnan(m.lm_head.weight.grad).any()


@pytest.mark.parametrize("bad", [dict(clip_low=1.5), dict(clip_low=-0.1), dict(clip_high=-0.1), dict(clip_high=float("inf")),
                                 dict(clip_low=float("nan")), dict(kl_coef=float("inf")), dict(beta=float("nan")),
                                 dict(label_smoothing=1.5), dict(label_smoothing=-0.5)])
def test_numbers_the_kernels_refuse_are_refused_on_the_plain_path(bad):
    idx, tgt, old, ref, adv = batch()
    m = plain(torch.float32)
    with pytest.raises(ValueError, match=next(iter(bad))):
        if "beta" in bad or "label_smoothing" in bad:
            m.preference_loss(idx, tgt, ref_logp=ref, **bad)
        else:
            m.policy_loss(idx, tgt, old, adv, ref_logp=ref, **bad)


def outlier_model(size, recompute=False):
    """The fused model with one channel of the residual stream ``size`` times the others' size."""
    m, flat = fused(recompute=recompute, act_bits=8)
    with torch.no_grad():
        m.tr.wpe.weight[:, 5] = size * 0.03
        m.tr.wte.weight[:, 5] = 0.0
    return m


@pytest.mark.parametrize("recompute", [False, True])
def test_8_bits_warn_of_an_outlier_channel(monkeypatch, recompute):
    """A channel 300 times its neighbours leaves them without digits: the first training forward says so, once; models
    without one, and scoring, say nothing."""
    import warnings

    post_emulation.emulate(monkeypatch)
    idx, tgt, _, _, _ = batch()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        outlier_model(1.0, recompute).token_logprobs(idx, tgt)
        m = outlier_model(300.0, recompute)
        with torch.no_grad():
            m.token_logprobs(idx, tgt)
    with pytest.warns(UserWarning, match=r"block 0 " + ("input" if recompute else "LayerNorm") + r": 12[0-9]"):
        first = m.token_logprobs(idx, tgt)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        assert torch.equal(m.token_logprobs(idx, tgt), first)


@pytest.mark.parametrize("size,least,most", [(1.0, 0.0, 0.02), (50.0, 0.13, 0.16), (300.0, 0.85, 0.96)])
def test_an_outlier_channel_takes_its_neighbours_digits(size, least, most):
    """What the format does to the other 127 channels of a block whose first is ``size`` standard deviations: a step of
    2^-5 at 2.7 of them (normal values), of 2^-1 at 50, of 4 at 300. Values are off by step / sqrt(12), 0.9% and 14%; at
    300 all that lie below 2 become 0, 95% of them with 74% of the squares (86% of the root mean square), and the others 4,
    off by at most 2 (96%)."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(400, 128, generator=g)
    x[:, 0] *= size
    if size > 1:
        x[:, 0] = size
    codes, e = post_emulation.act8_pack(x)
    off = (post_emulation.act8_unpack(codes, e, torch.float32) - x)[:, 1:]
    assert least <= off.norm() / x[:, 1:].norm() <= most
