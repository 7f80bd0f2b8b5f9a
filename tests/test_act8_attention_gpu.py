"""Attention backward from 8-bit Q/K/V on the GPU, at scores as sharp as a trained model's."""
import pytest
import torch

import act8_attention as A

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("amp", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("drop", [None, 0.2])
@pytest.mark.parametrize("offset", [0.0, 20.0, 40.0])
def test_backward_of_the_restored_scores(monkeypatch, offset, drop, amp):
    from heiretsu_b200.ops._C import check_status

    err, bound = A.error(monkeypatch, offset, "cuda", amp, drop)
    torch.cuda.synchronize()
    check_status()
    assert err <= bound, (err, bound)
