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
