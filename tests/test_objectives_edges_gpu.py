"""Post-training objectives on the GPU where a training program can go wrong (see test_objectives_edges_cpu.py)."""
import gc

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _leave_no_garbage():
    yield
    gc.collect()


def test_a_derivative_that_is_infinite_at_ignored_tokens():
    """sqrt(-logp): infinite at the 0 of ignored tokens, which torch.where leaves out. Gradients follow the plain path's
    (tolerance of the 16-bit heads)."""
    from heiretsu_b200.ops._C import check_status
    from test_objectives_gpu import IGNORE, batch, close, grads, models

    plain, fz = models()
    idx, tgt = batch()[:2]
    for m in (plain, fz):
        lp = m.token_logprobs(idx, tgt)
        (torch.where(tgt != IGNORE, (-lp).sqrt(), 0.0).sum() / 300).backward()
    torch.cuda.synchronize()
    check_status()
    close(grads(fz), grads(plain), 5e-2)


def test_fp16_probabilities_keep_their_gradient():
    from heiretsu_b200.ops._C import check_status
    from test_objectives_edges_cpu import check_fp16_range, fp16_range

    out = fp16_range("cuda", torch.float16)
    torch.cuda.synchronize()
    check_status()
    check_fp16_range(*out)


def test_balance_loss_beside_the_log_probabilities():
    """Fused mixture of experts: adding the aux loss changes the routers' gradient, in the way ``policy_loss`` returns it."""
    from heiretsu_b200.ops._C import check_status
    from test_objectives_gpu import batch, grads, models

    m = models(moe=True)[1]
    idx, tgt, adv = batch()[:3]
    out = []
    for weight in (0.0, 1.0):
        for p in m.parameters():
            p.main_grad.zero_()
        lp, aux = m.token_logprobs(idx, tgt, return_aux=True)
        ((lp * adv).sum() / 300 + weight * aux).backward()
        out.append(grads(m))
    with torch.no_grad():
        _, want, _, _ = m.policy_loss(idx, tgt, lp.detach(), adv)
    torch.cuda.synchronize()
    check_status()
    assert aux > 0 and abs(aux.item() - want.item()) <= 2.0 ** -20 * want.item()
    routers = [n for n in out[0] if "router" in n or "gate" in n]
    assert routers and all((out[1][n] - out[0][n]).norm() > 0 for n in routers)


@pytest.mark.parametrize("kl", [0.0, 0.1])
def test_policy_terms_past_32_bits(kl):
    """The kernel on ratios and KL terms that overflow 32 bits but take no part, against 64 bits."""
    from heiretsu_b200.ops import kernels as K
    from heiretsu_b200.ops._C import check_status
    from post_oracle import grad_bound, logprobs, lse_bound, policy
    from test_objectives_edges_cpu import overflowing

    V, n = 1000, 24
    _, old, adv, ref, w = overflowing(n, "cuda")
    if kl == 0:
        ref[15] = 300.0  # counts, in the statistic alone
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(n, V, device="cuda", generator=g)
    t = torch.randint(0, V, (n,), device="cuda", generator=g)
    lp64, lse64, unit = logprobs(x, V, t)
    near = (old + 300).abs() > 1  # the others' ratios go by the log-probability
    old = torch.where(near, (lp64 - 0.05).float(), old)
    ref = torch.where(ref < 100, (lp64 + 0.1).float(), ref)
    loss, stats, logp, grad = K.policy_loss(x, V, t, old, adv, ref_logp=ref, weights=w, clip_high=0.25, kl_coef=kl)
    torch.cuda.synchronize()
    check_status()
    live = torch.ones(n, dtype=torch.bool, device="cuda")
    want, wstats, d = policy(lp64, live, old, adv, ref, w, 0.2, 0.25, kl)
    slack = 2 * lse_bound(lse64, V).max().item() + 16 * 2.0 ** -24  # of a ratio, relative
    assert abs(loss.item() - want.item()) <= 2 * 1.3 * slack
    assert stats[1] == wstats[1].float()
    assert (torch.isinf(stats[0]) if kl == 0 else abs(stats[0].item() - wstats[0].item()) <= slack)
    assert torch.isfinite(grad).all() and (grad[9:15] == 0).all()  # weight 0; the others keep their KL term
    tol = grad_bound(d[:, None] * unit, d, x, lse64, V, x.dtype) + slack * (d[:, None] * unit).abs()
    assert ((grad.double() - d[:, None] * unit).abs() <= tol).all()


@pytest.mark.parametrize("P,T", [(16, 1), (17, 1), (32, 4), (16, 128), (17, 128), (8, 129), (9, 129), (1, 2049), (2, 2049),
                                 (4096, 1), (5000, 0), (1024, 4)])
def test_preference_pairs_on_both_sides_of_the_launch_rule(P, T):
    """One CTA takes as many pairs as it has groups of warps (16 up to 128 tokens, then halves); loss, rewards and gradient
    against 64 bits around that number. Only the outputs' roundings remain."""
    from heiretsu_b200.ops import kernels as K
    from heiretsu_b200.ops._C import check_status
    from post_oracle import IGNORE, preference

    g = torch.Generator(device="cuda").manual_seed(P + T)
    lp = -torch.rand(2 * P, T, device="cuda", generator=g)
    t = torch.randint(0, 9, (2 * P, T), device="cuda", generator=g)
    t[torch.rand(2 * P, T, device="cuda", generator=g) < 0.3] = IGNORE
    loss, rewards, d = K.preference_loss(lp, t, beta=0.4, label_smoothing=0.1)
    torch.cuda.synchronize()
    check_status()
    l64, r64, d64 = preference(lp, t, None, 0.4, 0.1)
    for a, b in ((loss, l64), (rewards, r64), (d, d64)):
        assert ((a.double() - b).abs() <= 2.0 ** -24 * b.abs() + 1e-12).all()


def test_many_short_preference_pairs_spread_over_the_gpu():
    """4096 pairs of one token are no queue on one SM: within 20 times of 16 pairs (in one CTA they took 160 times as long,
    on all SMs 2 times)."""
    from heiretsu_b200.ops import kernels as K

    def us(P):
        lp = -torch.rand(2 * P, 1, device="cuda")
        t = torch.zeros(2 * P, 1, device="cuda", dtype=torch.long)
        K.preference_loss(lp, t)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(10):
                K.preference_loss(lp, t)
        times = []
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            graph.replay()
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    assert us(4096) <= 20 * us(16)
