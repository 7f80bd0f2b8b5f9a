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
