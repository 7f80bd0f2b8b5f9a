"""Token log-probabilities, the clipped policy loss and the preference loss against 64-bit oracles.

Tolerances are derived in tests/post_oracle.py before any run: they count the roundings of the output, of the
exponentials and of the sums.
"""
import gc

import pytest
import torch

from post_oracle import EPS, IGNORE, grad_bound, logprobs, lse_bound, policy, preference

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


def make(M, V, W, dt, seed=0, off=0, ignored=0.25, ld=None):
    """Logits [M, W] (columns V.. hold NaN: nothing may read them) whose rows start `off` elements into a wider
    buffer of row stride `ld`, and targets with some rows ignored."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ld = ld or W + off
    buf = torch.full((max(M, 1), ld), float("nan"), device="cuda", dtype=dt)
    x = buf[:M, off:off + W]
    t = torch.randint(0, V, (M,), device="cuda", generator=g)
    v = 2 * torch.randn(M, V, device="cuda", generator=g)
    v.scatter_add_(1, t[:, None], 10 * torch.rand(M, 1, device="cuda", generator=g))
    x[:, :V] = v.to(dt)
    drop = torch.rand(M, device="cuda", generator=g) < ignored
    if M > 1:
        t[drop] = IGNORE
    return x, t, g


def copy_of(x, off):
    """A copy of `make`'s logits with the same layout (the order of a row's sum goes by its alignment)."""
    return x._base.clone()[:x.shape[0], off:off + x.shape[1]]


def check_rows(x, V, t, logp, lse, grad, coef):
    lp64, lse64, g64 = logprobs(x, V, t)
    b = lse_bound(lse64, V)
    assert ((logp.double() - lp64).abs() <= b + 4 * 2.0 ** -24 * lp64.abs()).all()
    if lse is not None:
        assert ((lse.double() - lse64).abs() <= b).all()
    if grad is not None:
        want = coef[:, None] * g64
        live = t != IGNORE
        assert (grad[~live] == 0).all()
        assert (grad[:, V:] == 0).all()
        tol = grad_bound(want, coef, x, lse64, V, x.dtype)
        assert ((grad[:, :V].double() - want).abs() <= tol)[live].all()


SHAPES = [  # M, V, W (row width), off (elements the rows are shifted by), ld
    (1, 1, 1, 0, None),
    (1, 7, 7, 0, None),
    (2, 8, 8, 0, None),
    (5, 129, 129, 0, None),
    (7, 1000, 1024, 0, None),
    (9, 1001, 1001, 3, 1009),     # rows that start on 2-byte (or 4-byte) boundaries only
    (6, 4096, 4096, 8, 4112),
    (33, 50257, 50304, 0, None),
    (300, 515, 520, 0, None),
    (700, 2049, 2056, 0, None),   # more rows than CTAs that run at once
    (2, 131071, 131071, 0, None),
    (1, 300001, 300001, 1, None),
    (160001, 33, 40, 0, None),    # more rows than one scan of the targets lists
]


@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("M,V,W,off,ld", SHAPES)
def test_token_logprobs(M, V, W, off, ld, dt):
    x, t, _ = make(M, V, W, dt, seed=M + V, off=off, ld=ld)
    keep = x.clone()
    logp, lse = K().token_logprobs(x, V, t)
    grad = torch.full((M + 1, W + 9), 7.0, device="cuda", dtype=dt)  # a guard row and guard columns
    logp2, lse2 = K().token_logprobs(x, V, t, grad=grad[:M, :W])
    status_ok()
    assert torch.equal(x.nan_to_num(5.0), keep.nan_to_num(5.0))
    one = (t != IGNORE).double()
    check_rows(x, V, t, logp, lse, None, None)
    check_rows(x, V, t, logp2, lse2, grad[:M, :W], one)
    assert (grad[M] == 7).all() and (grad[:, W:] == 7).all()
    inplace = copy_of(x, off)
    logp3, _ = K().token_logprobs(inplace, V, t, grad=inplace)
    assert torch.equal(logp3, logp2)
    assert torch.equal(inplace, grad[:M, :W])
    guard = inplace._base.clone()
    guard[:M, off:off + W] = float("nan")
    assert torch.isnan(guard).all()  # nothing beside the rows was written


def test_masked_logits():
    """Columns masked with -inf or the type's lowest value, rows with one or no column left, NaN and infinity in
    ignored rows."""
    for dt in (BF16, FP16, FP32):
        M, V = 8, 1003
        x, t, g = make(M, V, V, dt, seed=5, ignored=0.0)
        low = torch.finfo(dt).min
        x[0, 1:] = float("-inf")
        t[0] = 0                                     # one column left: logp 0, gradient 0
        x[1, torch.arange(V, device="cuda") != t[1]] = low
        x[2, ::2] = float("-inf")
        t[2] = 1
        x[3] = float("nan")
        t[3] = IGNORE
        x[4] = float("inf")
        t[4] = IGNORE
        x[5] = low                                   # all columns at the lowest value: uniform
        x[6, :900] = float("-inf")
        t[6] = 901
        grad = torch.empty_like(x)
        logp, lse = K().token_logprobs(x, V, t, grad=grad)
        status_ok()
        lp64, lse64, g64 = logprobs(torch.where(torch.isfinite(x) | (x == float("-inf")), x, torch.zeros_like(x)), V, t)
        tol = lse_bound(lse64, V)
        assert ((logp.double() - lp64).abs() <= tol).all(), (logp, lp64)
        assert (grad[3:5] == 0).all() and (logp[3:5] == 0).all() and (lse[3:5] == 0).all()
        assert (grad[0] == 0).all()
        assert (grad[2, ::2] == 0).all() and (grad[6, :900] == 0).all()
        for r in (1, 2, 5, 6, 7):
            assert ((grad[r].double() - g64[r]).abs() <= EPS[dt] * g64[r].abs() + 2e-5 + 2.0 ** -25).all(), r


@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("V,W,off", [(5003, 5008, 0), (70001, 70001, 3)])
def test_unlikely_targets(V, W, off, dt):
    """Targets far below the largest logit (80 to 1000), at -inf, or far above the rest; logits around 1e4."""
    M = 24
    x, t, _ = make(M, V, W, dt, seed=21, off=off, ignored=0.0)
    at = torch.arange(M, device="cuda")
    for r, low in enumerate((60, 80, 83, 85, 90, 120, 500, 1000)):
        x[r, t[r]] = -low
        x[r, (t[r] + 1) % V] = 2.0
    x[8, t[8]] = float("-inf")
    x[9, t[9]] = 60000.0 if dt == FP16 else 1e30
    x[10, :V] += 10000.0
    x[11, :V] -= 10000.0
    x[12, t[12]] = 200.0
    t[13] = IGNORE
    grad = torch.full_like(x, 3.0)
    logp, lse = K().token_logprobs(x, V, t, grad=grad)
    only, _ = K().token_logprobs(x, V, t)
    status_ok()
    assert torch.equal(only, logp)
    assert logp[8] == float("-inf") and torch.isfinite(lse).all()
    lp64, lse64, g64 = logprobs(x, V, t)
    ok = at != 8
    # the sum's own error, and roundings of log-probabilities of this size (fp32 x - lse at 1e4: 2^-24 of x, too)
    big = torch.where(torch.isfinite(x[at, t.clamp_min(0)]), x[at, t.clamp_min(0)].double().abs(), 0)
    tol = lse_bound(torch.zeros_like(lse64), V) + 8 * 2.0 ** -24 * lp64.abs() + 2.0 ** -24 * big
    assert ((logp.double() - lp64).abs() <= tol)[ok].all()
    assert ((lse.double() - lse64).abs() <= tol + 4 * 2.0 ** -24 * lse64.abs())[ok].all()
    assert (grad[13] == 0).all() and (grad[:, V:] == 0).all()
    rel = 2.0 ** -20 + tol[:, None]  # exponentials of arguments up to ~25 that matter, and the sum's error
    p = -g64
    p[at, t.clamp_min(0)] += 1.0     # p's error is the gradient's: 1 - p_t keeps no relative accuracy at p_t = 1
    assert ((grad[:, :V].double() - g64).abs() <= EPS[dt] * g64.abs() + rel * (p.abs() + 2.0 ** -24) + 2.0 ** -25).all()


def test_rows_without_any_value():
    """A counted row of -inf only, or with NaN or +inf, gives NaN (as a log-softmax does) and leaves the others alone."""
    M, V = 6, 777
    x, t, _ = make(M, V, V, FP32, seed=9, ignored=0.0)
    clean = x.clone()
    x[1] = float("-inf")
    x[2, 5] = float("nan")
    x[3, 700] = float("inf")
    grad = torch.empty_like(x)
    logp, _ = K().token_logprobs(x, V, t, grad=grad)
    want = torch.log_softmax(x, 1).gather(1, t[:, None])[:, 0]
    status_ok()
    assert torch.isnan(logp[1:4]).all() and torch.isnan(want[1:4]).all()
    assert torch.isnan(grad[1:4]).any(1).all()
    ref, _ = K().token_logprobs(clean, V, t)
    for r in (0, 4, 5):
        assert logp[r] == ref[r]


def test_bad_targets_are_reported():
    from heiretsu_b200.ops._C import check_status
    x, t, _ = make(4, 100, 104, BF16, seed=3, ignored=0.0)
    t[1], t[2] = 100, -7
    grad = torch.empty_like(x)
    logp, _ = K().token_logprobs(x, 100, t, grad=grad)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="bad argument"):
        check_status()
    assert torch.isnan(logp[1:3]).all() and torch.isfinite(logp[[0, 3]]).all()
    assert torch.isnan(grad[1:3, :100]).all() and torch.isfinite(grad[[0, 3]]).all()


def test_other_ignore_index_and_no_rows():
    x, t, _ = make(12, 64, 64, FP32, seed=4, ignored=0.0)
    t[3] = 0
    t2 = torch.where(t == 0, torch.full_like(t, IGNORE), t)
    a, _ = K().token_logprobs(x, 64, t, ignore_index=0)
    b, _ = K().token_logprobs(x, 64, t2)
    assert torch.equal(a, b)
    none = torch.full_like(t, IGNORE)
    loss, stats, logp, grad = K().policy_loss(x, 64, none, a, a, ref_logp=a)
    assert loss.item() == 0 and (stats == 0).all() and (logp == 0).all() and (grad == 0).all()
    e = torch.empty(0, 64, device="cuda")
    lp, lse = K().token_logprobs(e, 64, t[:0], grad=torch.empty_like(e))
    assert lp.numel() == 0 and lse.numel() == 0
    loss, stats, _, grad = K().policy_loss(e, 64, t[:0], lp, lp)
    assert loss.item() == 0 and grad.shape == (0, 64)
    status_ok()


@pytest.mark.parametrize("M,V,W", [(3, 50257, 50304), (61, 50257, 50304), (400, 5000, 5000)])
def test_scoring_and_losses_agree_bit_for_bit(M, V, W):
    """The same logits give the same log-probabilities with and without a gradient and in the policy loss, so the
    first policy step on freshly scored tokens has ratios of exactly 1: loss = -mean(A), nothing clipped, KL 0."""
    x, t, g = make(M, V, W, BF16, seed=M)
    score, _ = K().token_logprobs(x, V, t)
    again, _ = K().token_logprobs(x, V, t, grad=torch.empty_like(x))
    adv = torch.randn(M, device="cuda", generator=g)
    loss, stats, logp, _ = K().policy_loss(x, V, t, score, adv, ref_logp=score, kl_coef=0.5)
    status_ok()
    assert torch.equal(score, again) and torch.equal(score, logp)
    live = (t != IGNORE).double()
    want = -(live * adv.double()).sum() / live.sum()
    assert (stats == 0).all() and (loss.double() - want).abs() <= 2.0 ** -22 * (adv.abs().mean() + want.abs())


def policy_inputs(x, V, t, g, ref=True):
    """Log-ratios that keep at least 0.01 from the borders of the clip range (1 +- 0.2 .. 0.3 in ratio)."""
    M = t.numel()
    lp = logprobs(x, V, t)[0]
    far = torch.rand(M, device="cuda", generator=g) < 0.3
    side = torch.where(torch.rand(M, device="cuda", generator=g) < 0.5, -1.0, 1.0)
    d = torch.where(far, side * (0.4 + torch.rand(M, device="cuda", generator=g)),
                    (0.05 * torch.randn(M, device="cuda", generator=g)).clamp(-0.15, 0.15))
    old = (lp - d).float()
    adv = torch.randn(M, device="cuda", generator=g)
    return old, adv, (lp + 0.5 * torch.randn(M, device="cuda", generator=g)).float() if ref else None


def check_policy(x, V, t, old, adv, ref, weights, lo, hi, kl, scale, got):
    loss, stats, logp, grad = got
    live = t != IGNORE
    lp64, lse64, g64 = logprobs(x, V, t)
    l64, s64, d64 = policy(lp64, live, old, adv, ref, weights, lo, hi, kl)
    # logp's error enters every exponential as a relative error; the factors of e^d are at most e^1.5
    w = live.double() / live.sum().clamp_min(1) if weights is None else weights.double().abs() * live
    A = adv.double().repeat_interleave(t.numel() // adv.numel()).abs()
    rel = (lse_bound(lse64, V) + 4 * 2.0 ** -24 * (lp64.abs() + old.double().abs())).max() + 8 * 2.0 ** -24
    r = torch.exp((lp64 - old.double()) * live)
    u = torch.exp((ref.double() - lp64) * live) if ref is not None else torch.zeros_like(r)
    slack = rel * (r * A + kl * (u + 1))
    assert (loss.double() - l64).abs() <= (w * slack).sum() + 2.0 ** -24 * l64.abs() + 1e-30
    assert (stats[0].double() - s64[0]).abs() <= rel * (w * (u + 1)).sum() + 1e-30
    assert (stats[1].double() - s64[1]).abs() <= 2.0 ** -22 * s64[1] + 1e-30
    s = 1.0 if scale is None else scale.double().item()
    coef = d64 * s
    b = lse_bound(lse64, V)
    assert ((logp.double() - lp64).abs() <= b + 4 * 2.0 ** -24 * lp64.abs()).all()
    want = coef[:, None] * g64
    tol = grad_bound(want, coef, x, lse64, V, x.dtype) + (s * w * slack)[:, None] * g64.abs()
    assert ((grad[:, :V].double() - want).abs() <= tol)[live].all()
    assert (grad[~live] == 0).all() and (grad[:, V:] == 0).all()


@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("M,V,W,off,ld", SHAPES)
def test_policy_loss(M, V, W, off, ld, dt):
    x, t, g = make(M, V, W, dt, seed=2 * M + V, off=off, ld=ld)
    old, adv, ref = policy_inputs(x, V, t, g)
    wt = torch.rand(M, device="cuda", generator=g)
    wt[M // 2] = 0
    # fp16 gradients of small weights would be subnormal: a loss scale, as fp16 training has
    scale = torch.full((1,), 256.0 if dt == FP16 else 0.5, device="cuda")
    for kw in (dict(ref=ref, weights=None, lo=0.2, hi=0.28, kl=0.05, scale=scale),
               dict(ref=None, weights=wt, lo=0.25, hi=0.2, kl=0.3, scale=None)):
        got = K().policy_loss(x, V, t, old, adv, ref_logp=kw["ref"], weights=kw["weights"], clip_low=kw["lo"],
                              clip_high=kw["hi"], kl_coef=kw["kl"], grad_scale=kw["scale"])
        status_ok()
        check_policy(x, V, t, old, adv, kw["ref"], kw["weights"], kw["lo"], kw["hi"], kw["kl"], kw["scale"], got)
        again = copy_of(x, off)
        l2, s2, lp2, g2 = K().policy_loss(again, V, t, old, adv, ref_logp=kw["ref"], weights=kw["weights"],
                                          clip_low=kw["lo"], clip_high=kw["hi"], kl_coef=kw["kl"],
                                          grad_scale=kw["scale"], grad=again)
        assert torch.equal(l2, got[0]) and torch.equal(s2, got[1]) and torch.equal(lp2, got[2])
        assert torch.equal(g2, got[3]) and g2.data_ptr() == again.data_ptr()


def test_policy_advantage_per_sequence():
    """One advantage for each run of rows equals the same advantage given for every row."""
    x, t, g = make(24, 333, 336, BF16, seed=8)
    old, adv, ref = policy_inputs(x, 333, t, g)
    for n in (1, 4, 24):
        a = K().policy_loss(x, 333, t, old, adv[:n].contiguous(), ref_logp=ref, kl_coef=0.1)
        b = K().policy_loss(x, 333, t, old, adv[:n].repeat_interleave(24 // n), ref_logp=ref, kl_coef=0.1)
        for p, q in zip(a, b):
            assert torch.equal(p, q)


def test_policy_with_broken_inputs():
    """NaN or infinite log-probabilities and advantages reach their own row's gradient only, never the padding."""
    M, V, W = 10, 1001, 1024
    x, t, g = make(M, V, W, BF16, seed=14, ignored=0.0)
    old, adv, ref = policy_inputs(x, V, t, g)
    clean = K().policy_loss(x, V, t, old, adv, ref_logp=ref, kl_coef=0.1)
    old[1], adv[2], adv[3], ref[4] = float("nan"), float("inf"), float("nan"), float("inf")
    old[5] = float("inf")          # ratio 0: gradient 0 but for the KL term
    loss, stats, logp, grad = K().policy_loss(x, V, t, old, adv, ref_logp=ref, kl_coef=0.1)
    status_ok()
    assert not torch.isfinite(loss) and torch.equal(logp, clean[2])
    assert (grad[:, V:] == 0).all()
    for r in (0, 6, 7, 8, 9):
        assert torch.equal(grad[r], clean[3][r])
    assert not torch.isfinite(grad[1:5, :V]).all(1).any() and torch.isfinite(grad[5]).all()


def test_policy_gradient_against_differences():
    """fp32 logits: central differences of the kernel's own loss along random directions. Step h: the loss's rounding
    gives 2^-22 |loss| / h, the third derivative (at most ~10 for |A|, ratios and weights of this size) h^2 * 10."""
    M, V, h = 6, 50, 2.0 ** -6
    x, t, g = make(M, V, V, FP32, seed=12, ignored=0.2)
    old, adv, ref = policy_inputs(x, V, t, g)
    kw = dict(ref_logp=ref, clip_low=0.2, clip_high=0.2, kl_coef=0.1)
    loss, _, _, grad = K().policy_loss(x, V, t, old, adv, **kw)
    for k in range(4):
        v = torch.randn(M, V, device="cuda", generator=g)
        v /= v.norm()
        up = K().policy_loss(x + h * v, V, t, old, adv, **kw)[0].double()
        dn = K().policy_loss(x - h * v, V, t, old, adv, **kw)[0].double()
        num, ana = (up - dn) / (2 * h), (grad.double() * v).sum()
        assert (num - ana).abs() <= 4e-6 / h * (1 + loss.abs()) * 2 + 10 * h * h, (num, ana)


def pairs(P, T, seed, ref=True, empty=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randint(0, 100, (2 * P, T), device="cuda", generator=g)
    t[torch.rand(2 * P, T, device="cuda", generator=g) < 0.4] = IGNORE
    if empty and P:
        t[0] = IGNORE
        t[2 * P - 1] = IGNORE
    lp = -3 * torch.rand(2 * P, T, device="cuda", generator=g)
    r = lp + 0.3 * torch.randn(2 * P, T, device="cuda", generator=g) if ref else None
    return lp, t, r


@pytest.mark.parametrize("ref", [True, False])
@pytest.mark.parametrize("P,T", [(1, 1), (1, 57), (2, 128), (3, 1023), (5, 4097), (64, 33), (300, 7), (1, 20001), (1030, 2),
                                 (131, 1031), (1, 200001), (40000, 5)])
def test_preference_loss(P, T, ref):
    for beta, eps, empty in ((0.1, 0.0, False), (0.7, 0.1, True), (-0.2, 1.0, False)):
        lp, t, r = pairs(P, T, P + T, ref, empty)
        loss, rew, d = K().preference_loss(lp, t, ref_logp=r, beta=beta, label_smoothing=eps)
        status_ok()
        l64, r64, d64 = preference(lp, t, r, beta, eps)
        # sums run in 64 bits: only the outputs' roundings remain (and 64-bit ones, 1e-12 of the largest sum)
        scale = 1e-12 * (1 + r64.abs().max())
        assert (loss.double() - l64).abs() <= 2.0 ** -24 * l64.abs() + scale
        assert ((rew.double() - r64).abs() <= 2.0 ** -24 * r64.abs() + scale).all()
        assert ((d.double() - d64).abs() <= 2.0 ** -24 * d64.abs() + scale + 2.0 ** -149).all()
        assert (d[t == IGNORE] == 0).all()
        again = K().preference_loss(lp, t, ref_logp=r, beta=beta, label_smoothing=eps)
        assert all(torch.equal(a, b) for a, b in zip((loss, rew, d), again))


def test_preference_extremes():
    """Margins far beyond exp's range stay finite; NaN in ignored tokens is not read; NaN in a counted one shows."""
    lp, t, r = pairs(4, 16, 3, empty=False)
    t[:, 0] = 5
    lp[0, 0], lp[5, 0] = -1e6, -1e6
    lp[t == IGNORE] = float("nan")
    loss, rew, d = K().preference_loss(lp, t, ref_logp=r, beta=0.5)
    clean = torch.where(t == IGNORE, torch.zeros_like(lp), lp)
    l64, r64, d64 = preference(clean, t, r, 0.5)
    assert torch.isfinite(loss) and (loss.double() - l64).abs() <= 2.0 ** -23 * l64.abs()
    assert torch.isfinite(d).all() and ((d.double() - d64).abs() <= 2.0 ** -24 * d64.abs() + 1e-9).all()
    lp[2, 0] = float("nan")
    loss, rew, d = K().preference_loss(lp, t, ref_logp=r, beta=0.5)
    assert torch.isnan(loss) and torch.isnan(rew[0, 2]) and torch.isfinite(rew[:, [0, 1, 3]]).all()
    e = torch.empty(0, 5, device="cuda")
    loss, rew, d = K().preference_loss(e, e.long())
    assert loss.item() == 0 and rew.shape == (2, 0) and d.shape == (0, 5)
    z = torch.empty(4, 0, device="cuda")  # sequences without tokens: margin 0
    loss, rew, d = K().preference_loss(z, z.long())
    assert abs(loss.item() - 0.6931471805599453) <= 2.0 ** -24 and (rew == 0).all()
    status_ok()


def test_streams_and_graphs():
    """On another stream, captured and replayed with new inputs, and two graphs interleaved."""
    M, V = 40, 3000
    x, t, g = make(M, V, V, BF16, seed=31)
    old, adv, ref = policy_inputs(x, V, t, g)
    want = K().policy_loss(x, V, t, old, adv, ref_logp=ref, kl_coef=0.1)
    lp, pt, pr = pairs(6, 100, 4)
    pwant = K().preference_loss(lp, pt, ref_logp=pr)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = K().policy_loss(x, V, t, old, adv, ref_logp=ref, kl_coef=0.1)
        pgot = K().preference_loss(lp, pt, ref_logp=pr)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(pgot, pwant))
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = K().policy_loss(x, V, t, old, adv, ref_logp=ref, kl_coef=0.1)
            pout = K().preference_loss(lp, pt, ref_logp=pr)
        graphs.append((gr, out, pout))
    x.copy_(x.flip(0))
    want2 = K().policy_loss(x, V, t, old, adv, ref_logp=ref, kl_coef=0.1)
    for gr, _, _ in graphs * 2:
        gr.replay()
    torch.cuda.synchronize()
    for _, out, pout in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want2))
        assert all(torch.equal(a, b) for a, b in zip(pout, pwant))
    status_ok()


def test_two_streams_at_once():
    calls = []
    for k in range(4):
        x, t, g = make(64, 5000, 5000, BF16, seed=k)
        old, adv, ref = policy_inputs(x, 5000, t, g)
        calls.append((x, t, old, adv, ref, K().policy_loss(x, 5000, t, old, adv, ref_logp=ref, kl_coef=0.1)))
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    outs = [[] for _ in calls]
    for _ in range(5):
        for i, (st, c) in enumerate(zip(streams, calls)):
            with torch.cuda.stream(st):
                outs[i].append(K().policy_loss(c[0], 5000, c[1], c[2], c[3], ref_logp=c[4], kl_coef=0.1))
    torch.cuda.synchronize()
    for o, c in zip(outs, calls):
        for got in o:
            assert all(torch.equal(a, b) for a, b in zip(got, c[5]))


def test_refusals():
    x, t, g = make(8, 60, 64, BF16, seed=1)
    f = torch.zeros(8, device="cuda")
    tl, pl, pr = K().token_logprobs, K().policy_loss, K().preference_loss
    for call in (
            lambda: tl(x, 0, t), lambda: tl(x, 65, t), lambda: tl(x, 60, t[:7]), lambda: tl(x, 60, t.int()),
            lambda: tl(x.double(), 60, t), lambda: tl(x.t(), 8, t), lambda: tl(x[0], 60, t),
            lambda: tl(x, 60, t.cpu()), lambda: tl(x.cpu(), 60, t.cpu()), lambda: tl(x, 60, torch.stack([t, t], 1)[:, 0]),
            lambda: tl(x, 60, t, grad=x.float()), lambda: tl(x, 60, t, grad=torch.empty_like(x)[:, :59]),
            lambda: tl(x, 60, t, grad=torch.empty_like(x)[:7]),
            lambda: tl(x[:, :60], 60, t, grad=x[:, 1:61]),                  # overlaps the logits, shifted
            lambda: tl(x[:4], 60, t[:4], grad=x[1:5]),
            lambda: tl(x, 60, t, grad=torch.empty(1, 64, device="cuda", dtype=BF16).expand(8, 64)),
            lambda: pl(x, 60, t, f[:7], f), lambda: pl(x, 60, t, f, f[:3]), lambda: pl(x, 60, t, f, f[:0]),
            lambda: pl(x, 60, t, f.double(), f), lambda: pl(x, 60, t, f, f, ref_logp=f[:1]),
            lambda: pl(x, 60, t, f, f, weights=f.half()), lambda: pl(x, 60, t, f, f, clip_low=1.5),
            lambda: pl(x, 60, t, f, f, clip_high=-0.1), lambda: pl(x, 60, t, f, f, kl_coef=float("nan")),
            lambda: pl(x, 60, t, f, f, grad_scale=f), lambda: pl(x, 60, t, f, torch.zeros(1, device="cuda").expand(8)),
            lambda: pr(f.view(1, 8), t.view(1, 8)), lambda: pr(f, t), lambda: pr(f.view(2, 4), t.view(4, 2)[:1]),
            lambda: pr(f.view(2, 4).double(), t.view(2, 4)), lambda: pr(f.view(4, 2).t(), t.view(2, 4)),
            lambda: pr(f.view(2, 4), t.view(2, 4), ref_logp=f[:4]),
            lambda: pr(f.view(2, 4), t.view(2, 4), label_smoothing=1.2),
            lambda: pr(f.view(2, 4), t.view(2, 4), beta=float("inf")),
    ):
        with pytest.raises(RuntimeError):
            call()
    status_ok()
