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


def test_outlier_channels_are_reported_outside_of_captures():
    """The first training forward of an 8-bit model warns of a channel that takes its neighbours' digits, on a model whose
    first one is captured the first eager one; a captured step takes no host read."""
    import warnings

    from heiretsu_b200.ops._C import check_status
    from test_objectives_gpu import batch, models

    idx, tgt = batch()[:2]

    def outlier():
        m = models(act_bits=8)[1]
        with torch.no_grad():
            m.tr.wpe.weight[:, 5] = 9.0
        return m

    with warnings.catch_warnings():
        warnings.simplefilter("error")
        models(act_bits=8)[1].token_logprobs(idx, tgt).sum().backward()
    with pytest.warns(UserWarning, match="block 0 LayerNorm: 12[0-9]"):
        outlier().token_logprobs(idx, tgt).sum().backward()
    m = outlier()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with torch.cuda.graph(graph):
            m.token_logprobs(idx, tgt).sum().backward()
    graph.replay()
    with pytest.warns(UserWarning, match="block 0 LayerNorm"):
        m.token_logprobs(idx, tgt)
    torch.cuda.synchronize()
    check_status()


def test_column_sums_round_once_behind_the_ctas():
    """dgamma and dbeta of whole numbers: a CTA's sum of at most 2^6 rows of values below 2^18 is exact in 32 bits, the sum
    of all CTAs (2^30) only in 64, so what is added to the accumulators is off by its own rounding alone."""
    from heiretsu_b200.ops import kernels as K
    from heiretsu_b200.ops._C import check_status

    M, H = 8192, 1280
    g = torch.Generator(device="cuda").manual_seed(9)
    dy = torch.randint(2 ** 16, 2 ** 18, (M, H), device="cuda", generator=g).float()
    q = torch.ones(M, H, device="cuda", dtype=torch.int8)  # xh = 1 everywhere
    e = torch.full((M, H // 128), 127, device="cuda", dtype=torch.uint8)
    w, b, rstd = torch.ones(H, device="cuda"), torch.zeros(H, device="cuda"), torch.ones(M, device="cuda")
    res, d16 = torch.zeros(M, H, device="cuda"), torch.empty(M, H, device="cuda", dtype=torch.bfloat16)
    dg, db = torch.full((H,), 0.5, device="cuda"), torch.zeros(H, device="cuda")
    K.layernorm_bwd_act8(dy, q, e, rstd, w, b, res, res, d16, dg, db)
    torch.cuda.synchronize()
    check_status()
    want = dy.double().sum(0)
    assert torch.equal(db, want.float()) and torch.equal(dg, (want + 0.5).float())
