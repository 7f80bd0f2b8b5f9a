"""8-bit activations on inputs unlike random-initialised ones."""
import gc

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _leave_no_garbage():
    yield
    gc.collect()


@pytest.mark.parametrize("mean", [0.0, 10.0, 100.0, -300.0])
def test_layernorm_codes_of_rows_with_an_offset(mean):
    """The codes are those of the 64-bit value next to the middle between two codes as well, wherever the rows are
    centred. The second look has the mean to 2^-24 of the partial sums (at most 4 sqrt(H)) over H and rstd to 2^-46: xh to
    1e-8, 4e-7 of a step where 127 steps are 4 standard deviations, so about 8e-7 of the codes may differ; three times
    that, and 3 codes."""
    from heiretsu_b200.ops import kernels as K
    from heiretsu_b200.ops._C import check_status

    M, H = 2048, 1280
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(M, H, device="cuda", generator=g) + mean
    w, b = torch.ones(H, device="cuda"), torch.zeros(H, device="cuda")
    y, q, e, rstd = K.layernorm_fwd_act8(x, w, b)
    y0, _, rstd0 = K.layernorm_fwd(x, w, b)
    torch.cuda.synchronize()
    check_status()
    assert torch.equal(y, y0) and torch.equal(rstd, rstd0)
    xd = x.double()
    xh = (xd - xd.mean(1, keepdim=True)) * torch.rsqrt(xd.var(1, unbiased=False, keepdim=True) + 1e-5)
    block = torch.arange(H, device="cuda") // 128
    off = (q.double() != torch.round(xh * torch.exp2(127 - e.double())[:, block])).sum().item()
    assert off <= 3 * 8e-7 * M * H + 3, off
