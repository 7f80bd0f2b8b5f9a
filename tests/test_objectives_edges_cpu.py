"""Post-training objectives where a training program can go wrong: gradients that are infinite at positions that take no
part, values at the ends of a type's range, arguments that are refused. Plain path, and the fused path's host code on
stand-ins."""
import pytest
import torch

import post_emulation
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
