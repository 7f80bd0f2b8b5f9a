"""8-bit activations: the format against a 64-bit oracle (codes equal, values equal), and the LayerNorm that keeps
its normalised input in it."""
import gc

import pytest
import torch

from post_oracle import EPS, TINY, act8_codes, act8_values, gelu

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _leave_no_garbage():
    """Other tests count the memory held between two points: nothing of these may be freed in between."""
    yield
    gc.collect()

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def K():
    from heiretsu_b200.ops import kernels
    return kernels


def status_ok():
    from heiretsu_b200.ops._C import check_status
    torch.cuda.synchronize()
    check_status()


SHAPES = [(1, 1), (1, 16), (3, 127), (2, 128), (5, 129), (7, 256), (4, 500), (33, 1000), (257, 1280), (2, 8191), (3000, 40)]


def same_codes(x, q, e):
    codes, es, bad = act8_codes(x)
    assert torch.equal(torch.where(bad, torch.full_like(es, 255), es + 127), e.long())
    assert torch.equal(codes, q.long())
    return codes, es, bad


@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("M,N", SHAPES)
def test_pack_and_unpack(M, N, dt):
    g = torch.Generator(device="cuda").manual_seed(M * 10007 + N)
    x = (torch.randn(M, N, device="cuda", generator=g) * torch.exp2(torch.randint(-12, 8, (M, 1), device="cuda", generator=g))).to(dt)
    q, e = K().act8_pack(x)
    codes, es, bad = same_codes(x, q, e)
    for out in (BF16, FP16, FP32):
        y = K().act8_unpack(q, e, dtype=out)
        v = act8_values(codes, es, bad, out)
        assert torch.equal(y, v.to(out))  # a code times a power of two: exact, or one rounding where fp16 is subnormal
        h, y2 = K().act8_unpack_gelu(q, e, dtype=out)
        assert torch.equal(y, y2)
        want = gelu(v)
        # x / (1 + e^(-2u)): the exponential is off by 2 + 1.173 |2u| units, the rest by 8 roundings
        u = (0.7978845608028654 * (v + 0.044715 * v ** 3)).abs().clamp_max(50)
        rel = (4 + 2.4 * u) * 2.0 ** -23 + 8 * 2.0 ** -24
        assert ((h.double() - want).abs() <= (EPS[out] + rel) * want.abs() + TINY[out] + 1e-36).all()
    status_ok()


@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
def test_strided_rows(dt):
    """Rows that start at any element of a wider matrix; broadcast rows."""
    g = torch.Generator(device="cuda").manual_seed(1)
    base = torch.randn(9, 700, device="cuda", generator=g).to(dt)
    for off, n in ((1, 300), (3, 640), (8, 512), (4, 129)):
        x = base[:, off:off + n]
        q, e = K().act8_pack(x)
        same_codes(x, q, e)
    x = base[:1, :300].expand(9, 300)
    q, e = K().act8_pack(x)
    same_codes(x, q, e)
    status_ok()


@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("M,N", [(1, 128), (3, 128), (17, 384), (1001, 640), (64, 5120)])
def test_contiguous_and_strided_rows_give_the_same_codes(M, N, dt):
    """Whole blocks without a gap between rows are packed as one row; with a gap, or from an odd start, row by row."""
    g = torch.Generator(device="cuda").manual_seed(M + N)
    x = (torch.randn(M, N, device="cuda", generator=g) * torch.exp2(torch.randint(-12, 8, (M, 1), device="cuda", generator=g))).to(dt)
    x[M // 2, N - 1] = float("nan")
    x[M - 1, 0] = float("-inf")
    q, e = K().act8_pack(x)
    same_codes(x, q, e)
    for off, ld in ((0, N + 8), (1, N + 3)):
        wide = torch.full((M, ld), 1e4, device="cuda", dtype=dt)
        wide[:, off:off + N] = x
        q2, e2 = K().act8_pack(wide[:, off:off + N])
        assert torch.equal(q, q2) and torch.equal(e, e2)
    status_ok()


def test_extreme_values():
    for dt in (BF16, FP16, FP32):
        fi = torch.finfo(dt)
        rows = torch.zeros(12, 256, device="cuda")
        x = rows.to(dt)
        x[1, 3] = fi.max
        x[1, 130] = -fi.max
        x[2, 5] = fi.tiny
        x[3, 7] = fi.tiny * 2.0 ** -3   # subnormal
        x[4] = fi.max
        x[5, 0], x[5, 200] = float("inf"), 1.0
        x[6, 127], x[6, 128] = float("nan"), -2.0
        x[7, 1] = float("-inf")
        x[8] = 127.0
        x[9] = 127.0
        x[9, 64] = 128.0
        x[10] = 0.5
        x[10, 9] = 63.5                  # e = -1: halves are whole codes, nothing to round
        x[11, :128] = torch.arange(128, device="cuda") / 2  # ties
        x[11, 127] = 127.0
        q, e = K().act8_pack(x)
        codes, es, bad = same_codes(x, q, e)
        assert bad[5, 0] and not bad[5, 1] and bad[6, 0] and not bad[6, 1] and bad[7, 0]
        for out in (BF16, FP16, FP32):
            y = K().act8_unpack(q, e, dtype=out)
            v = act8_values(codes, es, bad, out).to(out)
            assert torch.equal(y.nan_to_num(12345.0), v.nan_to_num(12345.0))
            assert torch.isfinite(y[[1, 4]]).all() and torch.isnan(y[5, :128]).all() and y[5, 200] == 1
            h, _ = K().act8_unpack_gelu(q, e, dtype=out)
            assert torch.isnan(h[6, :128]).all() and torch.isfinite(h[6, 128:]).all()
            assert (h[1, 3] == y[1, 3]) and h[1, 130] == 0
    status_ok()


def test_error_is_within_half_a_code():
    x = torch.randn(512, 1024, device="cuda") * 3
    q, e = K().act8_pack(x)
    y = K().act8_unpack(q, e, dtype=FP32)
    top = x.abs().view(512, 8, 128).amax(2).repeat_interleave(128, 1)
    assert ((y - x).abs() <= top / 127).all()


def test_empty():
    for shape in ((0, 128), (4, 0), (0, 0)):
        q, e = K().act8_pack(torch.empty(shape, device="cuda"))
        assert q.shape == shape and K().act8_unpack(q, e).shape == shape
    status_ok()


def ln_inputs(M, H, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + M + H)
    x = torch.randn(M, H, device="cuda", generator=g) * 2 + 0.5
    w = 1 + 0.2 * torch.randn(H, device="cuda", generator=g)
    b = 0.3 * torch.randn(H, device="cuda", generator=g)
    return x, w, b, g


LN = [(1, 4), (2, 32), (5, 100), (9, 128), (17, 132), (64, 768), (300, 1024), (33, 1280), (1000, 1536), (12, 2048), (2500, 260)]


@pytest.mark.parametrize("f16", [BF16, FP16])
@pytest.mark.parametrize("M,H", LN)
def test_layernorm_forward(M, H, f16):
    x, w, b, _ = ln_inputs(M, H)
    y, q, e, rstd = K().layernorm_fwd_act8(x, w, b, 1e-5, dtype=f16)
    y0, mean0, rstd0 = K().layernorm_fwd(x, w, b, 1e-5, dtype=f16)
    status_ok()
    xd = x.double()
    mu = xd.mean(1, keepdim=True)
    r = torch.rsqrt((xd - mu).square().mean(1, keepdim=True) + 1e-5)
    xh = (xd - mu) * r
    # statistics: sums of H terms in 32 bits over 32 lanes: at most H / 32 + 8 roundings of values of |x|'s size
    rel = (H / 32 + 16) * 2.0 ** -24
    span = xd.abs().amax(1, keepdim=True) * r
    dxh = rel * (xh.abs() + span) + 4 * 2.0 ** -24 * xh.abs()
    assert ((rstd.double() - r[:, 0]).abs() <= 2 * rel * (1 + span[:, 0]) * r[:, 0]).all()
    want = xh * w.double() + b.double()
    assert ((y.double() - want).abs() <= EPS[f16] * want.abs() + TINY[f16] + dxh * w.double().abs() + 2.0 ** -23 * (want.abs() + b.abs())).all()
    # the codes are those of the 64-bit value; the exponent holds the row's block
    block = torch.arange(H, device="cuda") // 128
    step = torch.exp2(e.double() - 127)[:, block]
    assert ((q.double() * step - xh).abs() <= step / 2 + dxh).all()
    # (next to a border either code will do: rstd comes from H / 4 squares that are off by at most 6 * 2^-24 each,
    # rstd by half of that, and four standard deviations of their mean, of up to 127 steps, are left open)
    t = xh / step
    sure = ((t - t.floor()) - 0.5).abs() > 127 * 3 * 2.0 ** -24 * min(1, 4 / (H / 4) ** 0.5)
    assert torch.equal(q.double()[sure], torch.round(t)[sure])
    top = torch.zeros(M, e.shape[1], device="cuda", dtype=torch.float64)
    top.scatter_reduce_(1, block.expand(M, H), xh.abs(), "amax")
    full = 127 * torch.exp2(e.double() - 127)
    assert (top <= full * (1 + 1e-4)).all() and ((top > full / 2 * (1 - 1e-4)) | (e == 1)).all()
    assert torch.equal(rstd, rstd0) and torch.equal(y, y0)  # the forward pass does not change


@pytest.mark.parametrize("f16", [BF16, FP16])
@pytest.mark.parametrize("M,H", LN)
def test_layernorm_backward(M, H, f16):
    x, w, b, g = ln_inputs(M, H, seed=3)
    _, q, e, rstd = K().layernorm_fwd_act8(x, w, b, 1e-5, dtype=f16)
    dy = torch.randn(M, H, device="cuda", generator=g)
    dres_in = torch.randn(M, H, device="cuda", generator=g)
    block = torch.arange(H, device="cuda") // 128
    xh = q.double() * torch.exp2(e.double() - 127)[:, block]
    gw = dy.double() * w.double()
    m1, m2 = gw.mean(1, keepdim=True), (gw * xh).mean(1, keepdim=True)
    dx = rstd.double()[:, None] * (gw - m1 - xh * m2)
    want = dres_in.double() + dx
    # two means of H terms (H / 32 + 8 roundings of terms of this size), then six roundings
    rel = (H / 32 + 16) * 2.0 ** -24
    mag1, mag2 = gw.abs().mean(1, keepdim=True), (gw * xh).abs().mean(1, keepdim=True)
    tol = rstd.double()[:, None] * (rel * (mag1 + xh.abs() * mag2) + 6 * 2.0 ** -24 * (gw.abs() + m1.abs() + (xh * m2).abs())) \
        + 2 * 2.0 ** -24 * (want.abs() + dres_in.abs())
    outs = []
    for alias in (False, True):
        res = dres_in.clone()
        out = res if alias else torch.full((M, H), 9.0, device="cuda")
        o16 = torch.empty(M, H, device="cuda", dtype=f16)
        dg, db = torch.full((H,), 2.0, device="cuda"), torch.full((H,), -1.0, device="cuda")
        y = K().layernorm_bwd_act8(dy, q, e, rstd, w, b, res, out, o16, dg, db)
        outs.append((out.clone(), o16, dg, db, y))
    status_ok()
    for a, c in zip(*outs):
        assert torch.equal(a, c)
    out, o16, dg, db, y = outs[0]
    assert ((out.double() - want).abs() <= tol).all()
    assert torch.equal(o16, out.to(f16))
    n = (M / 8 + 64) * 2.0 ** -24  # column sums: at least 8 chains, then the partial rows
    for got, start, terms in ((dg, 2.0, dy.double() * xh), (db, -1.0, dy.double())):
        ref = start + terms.sum(0)
        assert ((got.double() - ref).abs() <= n * (abs(start) + terms.abs().sum(0)) + 2 * 2.0 ** -24 * ref.abs()).all()
    yw = xh * w.double() + b.double()
    assert ((y.double() - yw).abs() <= EPS[f16] * yw.abs() + TINY[f16] + 2.0 ** -23 * (yw.abs() + b.abs())).all()


def test_layernorm_gradient_against_differences():
    """Directional differences of sum(dy * LN(x)) in 64 bits at x; the codes are off by at most step / 2 per value, so
    dx = rstd (gw - m1 - xh m2) moves by at most rstd (step / 2) (|m2| + mean|gw|) per element (|xh| <= 4 taken
    with the mean's shift); the bound sums that along the direction."""
    M, H = 6, 256
    x, w, b, g = ln_inputs(M, H, seed=11)
    _, q, e, rstd = K().layernorm_fwd_act8(x, w, b, 1e-5)
    dy = torch.randn(M, H, device="cuda", generator=g)
    zero = torch.zeros(M, H, device="cuda")
    out, o16 = torch.empty_like(zero), torch.empty(M, H, device="cuda", dtype=BF16)
    dg, db = torch.zeros(2, H, device="cuda").unbind(0)
    K().layernorm_bwd_act8(dy, q, e, rstd, w, b, zero, out, o16, dg, db)
    f = lambda z: (dy.double() * torch.nn.functional.layer_norm(z, (H,), w.double(), b.double(), 1e-5)).sum()  # noqa: E731
    step = torch.exp2(e.double() - 127)[:, torch.arange(H, device="cuda") // 128]
    gw = (dy * w).double()
    xhmax = (q.double() * step).abs().amax(1, keepdim=True)
    slack = rstd.double()[:, None] * step / 2 * ((gw * q.double() * step).mean(1, keepdim=True).abs() + xhmax * gw.abs().mean(1, keepdim=True))
    for _ in range(3):
        v = torch.randn(M, H, device="cuda", generator=g).double()
        h = 1e-4
        num = (f(x.double() + h * v) - f(x.double() - h * v)) / (2 * h)
        ana = (out.double() * v).sum()
        assert (num - ana).abs() <= (slack * v.abs()).sum() + 1e-4, (num, ana)


def test_streams_graphs_and_nan():
    x, w, b, g = ln_inputs(200, 512)
    want = K().layernorm_fwd_act8(x, w, b)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y, q, e, r = K().layernorm_fwd_act8(x, w, b)
        q2, e2 = K().act8_pack(y)
        h, p = K().act8_unpack_gelu(q2, e2)
    gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip((y, q, e, r), want))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        h3, p3 = K().act8_unpack_gelu(*K().act8_pack(want[0]))
    s.synchronize()
    assert torch.equal(h, h3) and torch.equal(p, p3)
    x[3, 5] = float("nan")
    x[4, 6] = float("inf")
    y, q, e, r = K().layernorm_fwd_act8(x, w, b)
    assert (e[3:5] == 255).all() and torch.isnan(K().act8_unpack(q, e)[3:5]).all()
    assert torch.isfinite(y[[0, 1, 2, 5]]).all() and torch.isnan(y[3]).all()
    status_ok()


def test_refusals():
    x = torch.zeros(4, 256, device="cuda")
    w = torch.ones(256, device="cuda")
    q, e = K().act8_pack(x)
    ln, bw = K().layernorm_fwd_act8, K().layernorm_bwd_act8
    r = torch.ones(4, device="cuda")
    x16 = x.bfloat16()
    for call in (
            lambda: K().act8_pack(x.double()), lambda: K().act8_pack(x.t()), lambda: K().act8_pack(x.cpu()),
            lambda: K().act8_unpack(q, e[:, :1]), lambda: K().act8_unpack(q, e.int()), lambda: K().act8_unpack(q[:, :128], e[:, :1]),
            lambda: K().act8_unpack(q, e, dtype=torch.float64), lambda: K().act8_unpack(q, e.cpu()),
            lambda: ln(x16, w, w), lambda: ln(x, w[:255], w), lambda: ln(x, w, w, dtype=FP32), lambda: ln(x[:, :255].contiguous(), w[:255], w[:255]),
            lambda: ln(torch.zeros(2, 4096, device="cuda"), torch.ones(4096, device="cuda"), torch.ones(4096, device="cuda")),
            lambda: ln(x[:, :128], w[:128], w[:128]), lambda: ln(x, w.half(), w),
            lambda: bw(x, q, e, r[:3], w, w, x, x, x16, w, w), lambda: bw(x16, q, e, r, w, w, x, x, x16, w, w),
            lambda: bw(x, q, e, r, w, w, x, x, x, w, w), lambda: bw(x[:3], q, e, r, w, w, x, x, x16, w, w),
            lambda: bw(x, q, e, r, w, w, x, torch.zeros(2048, device="cuda")[:1024].view(4, 256).t().contiguous().t(), x16, w, w),
            lambda: (lambda z: bw(x, q, e, r, w, w, z[:1024].view(4, 256), z[4:1028].view(4, 256), x16, w, w))(
                torch.zeros(1100, device="cuda")),  # dres overlaps dres_in, shifted
            lambda: bw(x, q, e, r, w, w, x, x, x16, w, w.half()), lambda: bw(x, q, e, r, w, w, x, x[:, 1:], x16, w, w),
            lambda: bw(x, q, e, r, w, w, x, x, x16, w[:128], w),
    ):
        with pytest.raises(RuntimeError):
            call()
    status_ok()


def test_backward_refuses_one_buffer_for_both_parameter_gradients():
    x, w, b, g = ln_inputs(4, 256)
    _, q, e, r = K().layernorm_fwd_act8(x, w, b)
    dres, d16, sums = torch.zeros_like(x), x.bfloat16(), torch.zeros(512, device="cuda")
    for dg, db in ((sums[:256], sums[:256]), (sums[:256], sums[128:384]), (sums[200:456], sums[:256])):
        with pytest.raises(RuntimeError, match="dgamma and dbeta"):
            K().layernorm_bwd_act8(x, q, e, r, w, b, dres, dres, d16, dg, db)
    K().layernorm_bwd_act8(x, q, e, r, w, b, dres, dres, d16, sums[256:], sums[:256])  # next to each other
    status_ok()
