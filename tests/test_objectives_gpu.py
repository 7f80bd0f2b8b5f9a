"""Post-training objectives and 8-bit activations of the GPT model on the GPU: the fused path against the plain fp32
path, and the pieces together as a training program uses them (score with a frozen reference, preference or policy
step with 8-bit activations, AdamW, captured and replayed)."""
import gc

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _leave_no_garbage():
    """Other tests count the memory held between two points: nothing of these may be freed in between."""
    yield
    gc.collect()


IGNORE = -100
V, T = 1000, 256


def models(amp=torch.bfloat16, act_bits=16, recompute=False, dropout=0.0, n_layer=2, n_head=4, n_embed=256, moe=False):
    from heiretsu_b200.config import GPTConfig
    from heiretsu_b200.models.gpt import GPT
    from heiretsu_b200.parallel.flat import FlatParams

    kw = dict(num_experts=4, top_k=2, moe_freq=2) if moe else {}
    cfg = GPTConfig(block_size=T, vocab_size=V, n_layer=n_layer, n_head=n_head, n_embed=n_embed, dropout=dropout, **kw)
    out = []
    for fz in (False, True):
        torch.manual_seed(0)
        m = GPT(cfg).cuda()
        if fz:
            m.flat = FlatParams(m, torch.device("cuda"), dtype16=amp)
            m.fused, m.act_bits, m.recompute = True, act_bits, recompute
            if dropout > 0:
                seed = torch.tensor([99], dtype=torch.int32, device="cuda")
                for layer, blk in enumerate(m.tr.h):
                    blk._hb_dropout = (seed, layer, dropout)
        out.append(m)
    return out


def batch(n=4, seed=1, t=T):
    g = torch.Generator(device="cuda").manual_seed(seed)
    idx = torch.randint(0, V, (n, t), device="cuda", generator=g)
    tgt = torch.randint(0, V, (n, t), device="cuda", generator=g)
    for i in range(n):  # a prompt of its own length before the answer, padding behind
        tgt[i, :20 + 7 * i] = IGNORE
        tgt[i, t - 5 * i:] = IGNORE
    adv = torch.randn(n, t, device="cuda", generator=g)
    # log-ratios that 16-bit log-probabilities (off by about 0.02) do not carry across the clip range
    far = torch.rand(n, t, device="cuda", generator=g) < 0.3
    side = torch.where(torch.rand(n, t, device="cuda", generator=g) < 0.5, -1.0, 1.0)
    ratio = torch.where(far, side * 0.6, 0.05 * side)
    ref = 0.3 * torch.randn(n, t, device="cuda", generator=g)
    return idx, tgt, adv, ratio, ref


def grads(m):
    return {n: (p.main_grad if m.fused else p.grad).clone() for n, p in m.named_parameters()}


def close(a, b, tol):
    for n in b:
        rel = (a[n] - b[n]).norm().item() / (b[n].norm().item() + 1e-8)
        assert rel <= tol, (n, rel)


def objective(m, kind, b, base):
    idx, tgt, adv, ratio, ref = b
    if kind == "logp":
        lp = m.token_logprobs(idx, tgt)
        return (lp * adv).sum() / 300, lp
    if kind == "policy":
        loss, aux, stats, lp = m.policy_loss(idx, tgt, base - ratio, adv, ref_logp=base + ref, kl_coef=0.1)
        return loss + aux, lp
    loss, aux, rewards = m.preference_loss(idx, tgt, ref_logp=base + ref, beta=0.2)
    return loss + aux, rewards


@pytest.mark.parametrize("kind", ["logp", "policy", "preference"])
@pytest.mark.parametrize("amp", [torch.bfloat16, torch.float16])
def test_fused_against_plain(kind, amp):
    """Loss within 2e-2 and gradients within 5e-2 of the plain fp32 path: the tolerances of the cross-entropy head
    (the same operands in 16 bits)."""
    from heiretsu_b200.ops._C import check_status

    plain, fz = models(amp)
    b = batch()
    with torch.no_grad():
        base = plain.token_logprobs(b[0], b[1])
        assert (fz.token_logprobs(b[0], b[1]) - base).abs().max() < 0.1
    want, wrest = objective(plain, kind, b, base)
    want.backward()
    scale = 4096.0 if amp == torch.float16 else 1.0  # fp16 gradients need a loss scale, as in training
    if kind == "policy":
        fz.loss_grad_hint = scale if amp == torch.float16 else 0.5  # 0.5: the backward corrects it
    got, rest = objective(fz, kind, b, base)
    (scale * got).backward()
    torch.cuda.synchronize()
    check_status()
    assert abs(got.item() - want.item()) < 2e-2
    close({n: g / scale for n, g in grads(fz).items()}, grads(plain), 5e-2)
    assert (rest.float() - wrest.float()).abs().max() < (0.1 if kind != "preference" else 0.5)


def test_per_sequence_advantages_and_weights():
    plain, fz = models()
    idx, tgt, adv, ratio, _ = batch()
    w = torch.rand(4, T, device="cuda") / T
    with torch.no_grad():
        base = plain.token_logprobs(idx, tgt)
    for m in (plain, fz):
        a = m.policy_loss(idx, tgt, base - ratio, adv[:, 0], weights=w)
        c = m.policy_loss(idx, tgt, base - ratio, adv[:, :1].expand(4, T), weights=w)
        assert torch.equal(a[0], c[0])
    assert abs(a[0].item() - plain.policy_loss(idx, tgt, base - ratio, adv[:, 0], weights=w)[0].item()) < 2e-2


# The bound of tests/test_objectives_cpu.py (3.5% from the codes, doubled for the softmax's derivative), and twice the
# 16-bit path's own run-to-run spread (unordered reduce-adds), measured in place.
ACT8_TOL = 0.07


@pytest.mark.parametrize("recompute", [False, True])
@pytest.mark.parametrize("dropout,amp,moe", [(0.0, torch.bfloat16, False), (0.1, torch.bfloat16, False),
                                             (0.0, torch.float16, False), (0.0, torch.bfloat16, True)])
def test_act8_training_gradients(recompute, dropout, amp, moe):
    from heiretsu_b200.ops._C import check_status

    b = batch()
    tgt = b[1].clone()
    out = []
    for bits, rec in ((16, False), (16, False), (8, recompute)):
        _, m = models(amp, bits, rec, dropout, n_layer=3, moe=moe)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        _, loss, aux = m(b[0], tgt, return_logits=False)
        torch.cuda.synchronize()
        held = torch.cuda.memory_allocated() - before
        scale = 1024.0 if amp == torch.float16 else 1.0
        m.loss_grad_hint = scale
        (scale * (loss + aux)).backward()
        torch.cuda.synchronize()
        check_status()
        out.append((loss.item(), {n: g / scale for n, g in grads(m).items()}, held))
    (l0, g0, h0), (_, g0b, _), (l1, g1, h1) = out
    assert l0 == l1  # the forward pass does not change
    assert h1 < (0.6 if not moe else 0.9) * h0, (h1, h0)  # the logits (1000 columns) are held beside the blocks
    for n in g0:
        floor = (g0b[n] - g0[n]).norm().item()
        assert (g1[n] - g0[n]).norm().item() <= 2 * floor + ACT8_TOL * (g0[n].norm().item() + 1e-8), n


def test_preference_and_policy_training_together():
    """The operators as a run uses them: the frozen reference scores the batch, preference steps (8-bit activations,
    AdamW) leave the policy behind it, then a policy step on tokens scored by the policy itself."""
    from heiretsu_b200.ops._C import check_status
    from heiretsu_b200.optim import FusedAdamW

    _, ref = models()
    runs = []
    for bits in (16, 8):
        _, m = models(act_bits=bits)
        opt = FusedAdamW(m.flat, lr=1e-4, max_grad_norm=1.0)
        idx, tgt, adv, _, _ = batch(8)
        with torch.no_grad():
            ref_lp = ref.token_logprobs(idx, tgt)
        losses = []
        for _ in range(3):
            loss, _, rewards = m.preference_loss(idx, tgt, ref_logp=ref_lp, beta=0.5)
            loss.backward()
            opt.step()
            opt.zero_grad()
            losses.append(loss.item())
            if len(losses) == 1:  # the policy is the reference: no margin, log 2
                assert abs(losses[0] - 0.6931472) <= 2.0 ** -23 and (rewards == 0).all()
        with torch.no_grad():
            old = m.token_logprobs(idx, tgt)
        loss, _, stats, lp = m.policy_loss(idx, tgt, old, adv, ref_logp=ref_lp, kl_coef=0.02)
        assert torch.equal(lp.detach(), old) and stats[1] == 0 and stats[0] > 0
        live = (tgt != IGNORE).double()
        u = (ref_lp - old).double() * live
        want = (-(adv.double() * live).sum() + 0.02 * (torch.expm1(u) - u).sum()) / live.sum()
        assert abs(loss.item() - want.item()) < 1e-5
        loss.backward()
        opt.step()
        torch.cuda.synchronize()
        check_status()
        runs.append(losses)
    # the same curve with 8-bit activations: each step's move of the loss within twice the gradients' tolerance
    a, c = runs
    assert abs(a[0] - c[0]) < 1e-6
    assert abs((a[2] - a[0]) - (c[2] - c[0])) <= 2 * ACT8_TOL * abs(a[2] - a[0]) + 1e-3


@pytest.mark.parametrize("kind", ["policy", "preference"])
def test_captured_step_equals_eager(kind):
    """Forward and backward captured and replayed with new tokens, 8-bit activations; the run-to-run spread of the
    gradients (unordered fp32 reduce-adds) is the tolerance."""
    from heiretsu_b200.ops._C import check_status

    plain, m = models(act_bits=8)
    b1, b2 = batch(4, 1), batch(4, 2)
    with torch.no_grad():
        bases = [plain.token_logprobs(b[0], b[1]) for b in (b1, b2)]

    def eager(b, base):
        m.flat.grad.zero_() if hasattr(m.flat, "grad") else [p.main_grad.zero_() for p in m.parameters()]
        loss, _ = objective(m, kind, b, base)
        loss.backward()
        return loss.item(), grads(m)

    first = [eager(b, base) for b, base in zip((b1, b2), bases)]
    again = eager(b2, bases[1])
    static, sbase = [t.clone() for t in b1], bases[0].clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for p in m.parameters():
            p.main_grad.zero_()
        loss, _ = objective(m, kind, static, sbase)
        loss.backward()
    for (want, gw), b, base in zip(first, (b1, b2), bases):
        for s, t in zip(static, b):
            s.copy_(t)
        sbase.copy_(base)
        graph.replay()
        torch.cuda.synchronize()
        assert abs(loss.item() - want) <= 1e-6 * (1 + abs(want))
        for n, g in grads(m).items():
            floor = (again[1][n] - first[1][1][n]).norm().item()
            assert (g - gw[n]).norm().item() <= 4 * floor + 5e-3 * (gw[n].norm().item() + 1e-8), n
    check_status()


def test_engine_with_8_bit_activations():
    """--activation_bits 8 through the trainer: captured steps follow the 16-bit engine's first losses."""
    from heiretsu_b200.config import GPTConfig
    from heiretsu_b200.topo import init_topology
    from heiretsu_b200.trainer import Engine, build_argparser
    from heiretsu_b200.utils.data import SyntheticLoader

    curves = {}
    for bits, ck in ((16, 0), (8, 0), (8, 1)):
        args = build_argparser().parse_args([
            "--batch_size", "2", "--block_size", "256", "--grad_accum_steps", "2", "--n_layer", "2", "--n_head", "2",
            "--n_embed", "128", "--dropout", "0", "--amp", "bf16", "--engine", "fused", "--activation_bits", str(bits),
            "--activation_checkpointing", str(ck), "--learning_rate", "1e-4"])
        torch.manual_seed(0)
        cfg = GPTConfig(block_size=256, vocab_size=1000, n_layer=2, n_head=2, n_embed=128, dropout=0.0)
        eng = Engine(args, init_topology(dp=1), torch.device("cuda"), cfg)
        loader = SyntheticLoader(2, 256, 1000, seed=3)
        curves[bits, ck] = [float(eng.train_step(loader)[0].item()) for _ in range(5)]
        eng.close()
    base = curves[16, 0]
    for k in ((8, 0), (8, 1)):
        assert curves[k][0] == base[0]  # the forward pass does not change
        # AdamW's first steps move every weight by about the learning rate whatever the gradient's size: the curves part
        # by at most the loss's own movement
        for a, c in zip(curves[k][1:], base[1:]):
            assert abs(a - c) < 2e-2


def test_tensor_parallel_is_refused():
    _, m = models()

    class Topo:
        tp = 2

    m.topo = Topo()
    idx, tgt, adv, _, _ = batch()
    with pytest.raises(ValueError, match="tp 1"):
        m.token_logprobs(idx, tgt)
