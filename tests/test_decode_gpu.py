"""Decoding kernels against their definitions in 64 bits (tests/decode_oracle.py): the paged cache, attention of one new
token over it, and sampling."""
import math

import pytest
import torch

import decode_oracle as O

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _k():
    from heiretsu_b200.ops import kernels as K
    return K


def _status():
    from heiretsu_b200.ops._C import check_status
    check_status(torch.cuda.current_device())


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _same(a, b):
    """Equal values, NaN where the other has NaN."""
    return a.dtype == b.dtype and bool(((a == b) | (a.isnan() & b.isnan())).all())


def _slots(n, size, pages, g):
    order = torch.randperm(pages, device="cuda", generator=g)
    return (order[:, None] * size + torch.arange(size, device="cuda")).view(-1)[:n].contiguous()


# ---- the cache ---------------------------------------------------------------------
@pytest.mark.parametrize("dtype,bits", [(BF16, 8), (F16, 8), (BF16, 16), (F16, 16)])
@pytest.mark.parametrize("n,heads,dim,size", [(1, 12, 64, 64), (37, 3, 128, 16), (130, 5, 32, 48), (259, 1, 16, 32), (0, 2, 64, 16)])
def test_cache_round_trip(n, heads, dim, size, dtype, bits):
    K, g = _k(), _gen(n + dim)
    pages = n // size + 3
    c = O.Cache(pages, heads, size, dim, dtype, bits)
    # views of a projection's output; heads of unlike sizes, some of them all zero
    qkv = torch.randn(n, 3, heads, dim, device="cuda", generator=g) * torch.exp(4 * torch.randn(n, 3, heads, 1, device="cuda", generator=g))
    qkv[:: 7, 1] = 0
    qkv = qkv.to(dtype)
    k, v = qkv[:, 1], qkv[:, 2]
    slots = _slots(n, size, pages, g)
    if n > 5:
        slots[3] = -1
    before = {m: t.clone() for m, t in c.pools.items()}
    K.kv_write(k, v, slots, **c.pools)
    want = O.Cache(pages, heads, size, dim, dtype, bits)
    live = slots >= 0
    want.put(slots[live], k[live], v[live])
    for m in c.pools:  # every slot, those that were not written as they were
        assert torch.equal(c.pools[m].view(torch.uint8), want.pools[m].view(torch.uint8)), m
    assert n == 0 or not torch.equal(before["k_pages"].view(torch.uint8), c.pools["k_pages"].view(torch.uint8))
    for dt in (BF16, F16, F32) if bits == 8 else (dtype,):
        rk, rv = K.kv_read(slots, **c.pools, dtype=dt)
        for r, x in ((rk, k), (rv, v)):
            ref = c.kept(x).where(live[:, None, None], torch.zeros((), dtype=torch.float64, device="cuda"))
            if bits == 8:
                ref = ref.clamp(-torch.finfo(dt).max, torch.finfo(dt).max)
            same = _same(r, ref.to(dt))
            assert same
    _status()


def test_cache_reads_a_slot_twice_and_in_any_order():
    K, g = _k(), _gen(3)
    c = O.Cache(4, 2, 16, 64, BF16, 8)
    k, v = torch.randn(2, 64, 2, 64, device="cuda", generator=g).to(BF16).unbind(0)
    K.kv_write(k, v, torch.arange(64, device="cuda"), **c.pools)
    at = torch.tensor([5, 63, 5, 0, -1, 17], device="cuda")
    rk, rv = K.kv_read(at, **c.pools)
    for r, x in ((rk, k), (rv, v)):
        ref = O.act8_values(x)[0][at.clamp_min(0)]
        ref[4] = 0
        assert torch.equal(r, ref.to(BF16))


@pytest.mark.parametrize("offset", [0, 1, 3])
def test_cache_takes_rows_at_any_address(offset):
    """K and V that start at any 2-byte address, with any strides; a cache whose slots lie heads apart."""
    K, g = _k(), _gen(4)
    buf = torch.randn(50 * (3 * 4 * 32 + 5) + 8, device="cuda", generator=g).to(F16)
    qkv = buf[offset:].as_strided((50, 3, 4, 32), (3 * 4 * 32 + 5, 4 * 32, 32, 1))
    k, v = qkv[:, 1], qkv[:, 2]
    for bits in (8, 16):
        c = O.Cache(4, 4, 16, 32, F16, bits)
        # [pages, size, 2, heads, dim] in memory
        nat = torch.zeros(4, 16, 2, 4, 32, device="cuda", dtype=c.pools["k_pages"].dtype)
        c.pools["k_pages"], c.pools["v_pages"] = nat[:, :, 0].transpose(1, 2), nat[:, :, 1].transpose(1, 2)
        slots = _slots(50, 16, 4, g)
        K.kv_write(k, v, slots, **c.pools)
        rk, rv = K.kv_read(slots, **c.pools, dtype=F16)
        same = _same(rk, c.kept(k).to(F16)) and _same(rv, c.kept(v).to(F16))
        assert same


def test_cache_keeps_broken_heads_apart():
    """An infinity or NaN makes its own head of its own token NaN, and no other; the largest values stay finite."""
    K, g = _k(), _gen(5)
    k, v = torch.randn(2, 16, 2, 64, device="cuda", generator=g).to(BF16).unbind(0)
    k, v = k.clone(), v.clone()
    k[3, 1, 5], v[4, 0, 63], k[6, 0, 0] = math.inf, math.nan, torch.finfo(BF16).max
    c = O.Cache(1, 2, 16, 64, BF16, 8)
    K.kv_write(k, v, torch.arange(16, device="cuda"), **c.pools)
    for dt in (BF16, F16, F32):
        top = torch.finfo(dt).max
        rk, rv = K.kv_read(torch.arange(16, device="cuda"), **c.pools, dtype=dt)
        for r, x in ((rk, k), (rv, v)):
            same = _same(r, O.act8_values(x)[0].clamp(-top, top).to(dt))
            assert same


def test_cache_slots_behind_the_end_are_reported():
    K = _k()
    c = O.Cache(2, 1, 16, 16, BF16, 16)
    k = torch.ones(3, 1, 16, device="cuda", dtype=BF16)
    before = c.pools["k_pages"].clone()
    K.kv_write(k, k, torch.tensor([32, 2 ** 40, -5], device="cuda"), **c.pools)
    assert torch.equal(c.pools["k_pages"].view(torch.int16), before.view(torch.int16))
    with pytest.raises(RuntimeError, match="bad argument"):
        _status()
    K.kv_write(k, k, torch.tensor([0, 1, 2], device="cuda"), **c.pools)
    _status()
    r, _ = K.kv_read(torch.tensor([0, 32, 1], device="cuda"), **c.pools)
    assert torch.equal(r[::2], k[::2]) and bool(r[1].isnan().all())
    with pytest.raises(RuntimeError, match="bad argument"):
        _status()


# ---- attention ---------------------------------------------------------------------
def _batch(lengths, heads, kv, dim, size, dtype, bits, seed, spare=2, offset=0.0):
    """Queries and a filled cache: (q, cache, table, lengths, per sequence the K and V it holds)."""
    g = _gen(seed)
    B = len(lengths)
    need = [(n + size - 1) // size for n in lengths]
    pages, wide = sum(need) + spare, max(need + [1]) + 1
    order = torch.randperm(pages, device="cuda", generator=g).tolist()
    c = O.Cache(pages, kv, size, dim, dtype, bits)
    table = torch.full((B, wide), -7, dtype=torch.int32, device="cuda")
    held = []
    for b, n in enumerate(lengths):
        mine = torch.tensor([order.pop() for _ in range(need[b])], device="cuda", dtype=torch.long)
        table[b, : need[b]] = mine.int()
        k, v = torch.randn(2, n, kv, dim, device="cuda", generator=g).unbind(0)
        k = (k + offset).to(dtype)
        v = v.to(dtype)
        at = torch.arange(n, device="cuda")
        c.put(mine[at // size] * size + at % size, k, v)
        held.append((c.kept(k), c.kept(v)))
    q = (2 * torch.randn(B, heads, dim, device="cuda", generator=g)).to(dtype)
    return q, c, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), held


def _compare(out, lse, q, held, scale=None):
    D = q.shape[2]
    scale = D ** -0.5 if scale is None else scale
    for b, (k, v) in enumerate(held):
        want, wl, size, mean_v = O.attention(q[b], k, v, scale)
        near, near_lse = O.attention_bounds(want, torch.where(torch.isfinite(wl), wl, 0.0), size, mean_v, D, k.shape[0], q.dtype)
        if k.shape[0] == 0:
            assert bool((out[b] == 0).all()) and bool((lse[b] == -math.inf).all()), b
            continue
        far = ((out[b].double() - want).abs() / near).max()
        assert far <= 1, (b, k.shape[0], float(far))
        far = ((lse[b].double() - wl).abs() / near_lse).max()
        assert far <= 1, (b, k.shape[0], float(far))


HEADS = [(12, 12, 64), (4, 4, 128), (8, 2, 128), (5, 1, 64), (8, 8, 32), (6, 2, 16), (16, 1, 64), (24, 1, 32), (9, 1, 128)]


@pytest.mark.parametrize("dtype,bits", [(BF16, 16), (F16, 16), (BF16, 8), (F16, 8)])
@pytest.mark.parametrize("heads,kv,dim", HEADS)
def test_attention_of_ragged_batches(heads, kv, dim, dtype, bits):
    K = _k()
    lengths = [1, 0, 15, 16, 17, 64, 63, 130, 0, 2, 259, 31, 513]
    for size in (16, 48, 64):
        q, c, table, n, held = _batch(lengths, heads, kv, dim, size, dtype, bits, seed=heads + dim + size)
        out, lse = K.decode_attention(q, table=table, lengths=n, **c.pools)
        assert out.shape == q.shape and out.dtype == dtype and lse.dtype == F32
        _compare(out, lse, q, held)
    _status()


@pytest.mark.parametrize("heads,kv,dim,dtype,bits", [(8, 2, 64, BF16, 16), (4, 4, 128, F16, 8), (12, 12, 64, BF16, 8)])
@pytest.mark.parametrize("lengths", [[1], [57], [4099], [20011, 3], [1] * 300, [700] * 40, [0] * 5, [0, 0, 5000, 0]])
def test_attention_of_other_batches(lengths, heads, kv, dim, dtype, bits):
    """One token to a long cache, one sequence to many: every way the work is split."""
    K = _k()
    q, c, table, n, held = _batch(lengths, heads, kv, dim, 32, dtype, bits, seed=len(lengths) + heads)
    out, lse = K.decode_attention(q, table=table, lengths=n, **c.pools)
    _compare(out, lse, q, held)
    again, lse2 = K.decode_attention(q, table=table, lengths=n, **c.pools)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    _status()


@pytest.mark.parametrize("bits", [16, 8])
def test_attention_at_sharp_scores_and_with_a_scale(bits):
    """An offset common to K's channels and scores of a large spread: one token carries the row, or a few do."""
    K = _k()
    for scale in (None, 1.0, 0.01, 0.0, -0.3):
        q, c, table, n, held = _batch([300, 40, 2000], 4, 2, 64, 16, BF16, bits, seed=9, offset=5.0)
        out, lse = K.decode_attention(q, table=table, lengths=n, scale=scale, **c.pools)
        _compare(out, lse, q, held, scale)


def test_attention_strides_and_alignment():
    """Queries that are views of a projection's output at any 2-byte address, a table that is part of a wider one, and a cache
    whose slots lie heads apart."""
    K = _k()
    q, c, table, n, held = _batch([100, 33, 1, 260], 8, 4, 64, 32, BF16, 16, seed=2)
    for offset, pad in ((0, 0), (1, 0), (2, 4), (8, 8)):
        buf = torch.zeros(offset + 4 * (3 * 8 * 64 + pad), device="cuda", dtype=BF16)
        view = buf[offset:].as_strided((4, 8, 64), (3 * 8 * 64 + pad, 64, 1))
        view.copy_(q)
        out, lse = K.decode_attention(view, table=table, lengths=n, **c.pools)
        _compare(out, lse, q, held)
    wide = torch.full((4, table.shape[1] + 9), 2 ** 30, dtype=torch.int32, device="cuda")
    wide[:, 3:3 + table.shape[1]] = table
    nat = torch.empty(c.pools["k_pages"].shape[0], 32, 2, 4, 64, device="cuda", dtype=BF16)
    k, v = nat[:, :, 0].transpose(1, 2), nat[:, :, 1].transpose(1, 2)
    k.copy_(c.pools["k_pages"]), v.copy_(c.pools["v_pages"])
    out, lse = K.decode_attention(q, k, v, wide[:, 3:3 + table.shape[1]], n)
    _compare(out, lse, q, held)
    q2 = q.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    out, lse = K.decode_attention(q2, table=table, lengths=n, **c.pools)
    _compare(out, lse, q, held)
    assert out.is_contiguous()


def test_attention_of_infinities_and_nan_in_counted_tokens():
    """A NaN in a counted token reaches its own sequence's heads and no other's; scores that are all -inf give NaN as 0 / 0
    does; one that is -inf weighs nothing."""
    K = _k()
    q, c, table, n, held = _batch([40, 40, 40, 20], 2, 2, 64, 16, BF16, 16, seed=1)
    q = torch.ones_like(q)
    kp = c.pools["k_pages"]
    slot = lambda b, t: (int(table[b, t // 16]), t % 16)  # noqa: E731
    pg, at = slot(0, 17)
    kp[pg, 0, at, 3] = math.nan
    for t in range(40):
        pg, at = slot(1, t)
        kp[pg, 1, at, 0] = -math.inf
    pg, at = slot(2, 39)
    kp[pg, 0, at, 9] = -math.inf
    out, lse = K.decode_attention(q, table=table, lengths=n, **c.pools)
    assert bool(out[0, 0].isnan().all()) and bool(lse[0, 0].isnan())
    assert bool(out[1, 1].isnan().all())
    k, v = held[2]
    want, wl, size, mean_v = O.attention(q[2, :1], k[:39, :1], v[:39, :1], 0.125)
    near, _ = O.attention_bounds(want, wl, size, mean_v, 64, 39, BF16)
    assert bool(((out[2, 0].double() - want[0]).abs() <= near[0]).all())
    for b, h in ((0, 1), (1, 0), (2, 1), (3, 0), (3, 1)):
        k, v = held[b]
        want, wl, size, mean_v = O.attention(q[b, h:h + 1], k[:, h:h + 1], v[:, h:h + 1], 0.125)
        near, _ = O.attention_bounds(want, wl, size, mean_v, 64, k.shape[0], BF16)
        assert bool(((out[b, h].double() - want[0]).abs() <= near[0]).all()), (b, h)
    _status()


@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 64), (8, 2, 128)])
def test_attention_of_broken_heads_in_8_bits(heads, kv, dim):
    """A head of one token whose K or V held an infinity or NaN: NaN in the query heads that share it, in its own sequence, and
    nowhere else; heads of zeros, and scales far apart, are like any others."""
    K = _k()
    q, c, table, n, held = _batch([40, 33, 50, 64], heads, kv, dim, 16, BF16, 8, seed=3)
    held = [(k.clone(), v.clone()) for k, v in held]

    def put(b, tok, h, name, byte=None, zero=False):
        pg, at = int(table[b, tok // 16]), tok % 16
        i = 0 if name == "k" else 1
        if byte is not None:
            c.pools[name + "_exp"][pg, h, at] = byte
            held[b][i][tok, h] = math.nan
        if zero:
            c.pools[name + "_exp"][pg, h, at], c.pools[name + "_pages"][pg, h, at] = 1, 0
            held[b][i][tok, h] = 0

    put(0, 17, 1, "k", 255)
    put(1, 32, 0, "v", 255)
    for tok in range(50):
        put(2, tok, 0, "v", zero=True)
        put(2, tok, 1, "k", zero=True)
    pg, at = int(table[3, 0]), 5
    c.pools["v_exp"][pg, 0, at] += 30  # one token's V a billion times as large
    held[3][1][5, 0] *= 2.0 ** 30
    out, lse = K.decode_attention(q, table=table, lengths=n, **c.pools)
    G = heads // kv
    for b, (k, v) in enumerate(held):
        want, wl, size, mean_v = O.attention(q[b], k, v, dim ** -0.5)
        near, near_lse = O.attention_bounds(want, wl, size, mean_v, dim, k.shape[0], BF16)
        for h in range(heads):
            if (b, h // G) == (0, 1):
                assert bool(out[b, h].isnan().all()) and bool(lse[b, h].isnan())
            elif (b, h // G) == (1, 0):
                assert bool(out[b, h].isnan().all()) and abs(float(lse[b, h] - wl[h])) <= float(near_lse[h])
            else:
                assert bool(((out[b, h].double() - want[h]).abs() <= near[h]).all()), (b, h)
                assert abs(float(lse[b, h] - wl[h])) <= float(near_lse[h])
    _status()


@pytest.mark.parametrize("bits", [16, 8])
def test_attention_of_more_sequences_than_one_launch_takes(bits):
    K = _k()
    lengths = [(7 * i) % 40 for i in range(1030)] + [300, 0, 5]
    q, c, table, n, held = _batch(lengths, 2, 1, 32, 16, BF16, bits, seed=4)
    out, lse = K.decode_attention(q, table=table, lengths=n, **c.pools)
    _compare(out, lse, q, held)
    _status()


def test_attention_reports_bad_pages_and_lengths():
    K = _k()
    q, c, table, n, held = _batch([100, 33, 70, 260, 48], 4, 2, 64, 16, BF16, 16, seed=6)
    for where, what in (("table", c.pools["k_pages"].shape[0]), ("table", -1), ("lengths", -1), ("lengths", table.shape[1] * 16 + 1)):
        t, m = table.clone(), n.clone()
        if where == "table":
            t[3, 11] = what
        else:
            m[3] = what
        out, lse = K.decode_attention(q, table=t, lengths=m, **c.pools)
        assert bool(out[3].isnan().all()) and bool(lse[3].isnan().all())
        rest = [0, 1, 2, 4]
        _compare(out[rest], lse[rest], q[rest], [held[b] for b in rest])
        with pytest.raises(RuntimeError, match="bad argument"):
            _status()
    out, lse = K.decode_attention(q, table=table, lengths=n, **c.pools)
    _compare(out, lse, q, held)
    _status()


def test_attention_of_no_sequences_and_an_empty_table():
    K = _k()
    c = O.Cache(2, 2, 16, 64, BF16, 16)
    q = torch.ones(0, 4, 64, device="cuda", dtype=BF16)
    out, lse = K.decode_attention(q, table=torch.zeros(0, 3, dtype=torch.int32, device="cuda"),
                                  lengths=torch.zeros(0, dtype=torch.int32, device="cuda"), **c.pools)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    q = torch.ones(3, 4, 64, device="cuda", dtype=BF16)
    out, lse = K.decode_attention(q, table=torch.zeros(3, 0, dtype=torch.int32, device="cuda"),
                                  lengths=torch.zeros(3, dtype=torch.int32, device="cuda"), **c.pools)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    _status()


def test_attention_past_32_bit_offsets():
    """A cache of more than 2^31 elements: pages at its far end."""
    K, g = _k(), _gen(8)
    pages, size, kv, dim = 2 ** 31 // (64 * 2 * 128) + 40, 64, 2, 128
    pools = {n: torch.empty(pages, kv, size, dim, device="cuda", dtype=BF16) for n in ("k_pages", "v_pages")}
    q = torch.randn(2, 4, dim, device="cuda", generator=g).to(BF16)
    table = torch.tensor([[pages - 1, pages - 3, 5], [pages - 2, 0, pages - 9]], dtype=torch.int32, device="cuda")
    n = torch.tensor([150, 100], dtype=torch.int32, device="cuda")
    held = []
    for b in range(2):
        k, v = torch.randn(2, int(n[b]), kv, dim, device="cuda", generator=g).to(BF16).unbind(0)
        at = torch.arange(int(n[b]), device="cuda")
        slots = table[b].long()[at // size] * size + at % size
        K.kv_write(k, v, slots, **pools)
        rk, rv = K.kv_read(slots, **pools)
        assert torch.equal(rk, k) and torch.equal(rv, v)
        held.append((k.double(), v.double()))
    out, lse = K.decode_attention(q, table=table, lengths=n, **pools)
    _compare(out, lse, q, held)


def test_decoding_in_a_graph_and_on_other_streams():
    """Write, attention and sampling captured once and replayed as the sequences grow; two graphs and a stream of their own at
    the same time give what single calls give."""
    K, g = _k(), _gen(11)
    B, H, D, size, V = 6, 4, 64, 16, 1000
    wide = 8
    table = torch.randperm(B * wide, device="cuda", generator=g).int().view(B, wide)
    steps = 20
    k, v, q = torch.randn(3, steps, B, H, D, device="cuda", generator=g).to(BF16).unbind(0)
    logits = (4 * torch.randn(steps, B, V, device="cuda", generator=g)).to(BF16)
    u = torch.rand(steps, B, device="cuda", generator=g)
    start = torch.tensor([0, 3, 15, 16, 40, 100], dtype=torch.int32, device="cuda")

    def fresh():
        c = O.Cache(B * wide, H, size, D, BF16, 8)
        for b in range(B):
            m = int(start[b])
            at = torch.arange(m, device="cuda")
            gg = _gen(100 + b)
            kk, vv = torch.randn(2, m, H, D, device="cuda", generator=gg).to(BF16).unbind(0)
            c.put(table[b].long()[at // size] * size + at % size, kk, vv)
        return c

    def step(c, lengths, k, v, q, x, u):
        pos = lengths.long()
        slots = table.long().gather(1, (pos // size)[:, None])[:, 0] * size + pos % size
        K.kv_write(k, v, slots, **c.pools)
        lengths += 1
        out, lse = K.decode_attention(q, table=table, lengths=lengths, **c.pools)
        return out, lse, K.sample_tokens(x, V, u, temperature=0.8, top_k=50, top_p=0.9)

    single, lengths, want = fresh(), start.clone(), []
    for i in range(steps):
        want.append([t.clone() for t in step(single, lengths, k[i], v[i], q[i], logits[i], u[i])])
    graphs = []
    for _ in range(2):
        c, ln = fresh(), start.clone()
        ins = [t[0].clone() for t in (k, v, q, logits, u)]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(c, ln, *ins)  # warm-up outside the capture
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        c2 = fresh()
        for m in c.pools:
            c.pools[m].copy_(c2.pools[m])
        ln.copy_(start)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = step(c, ln, *ins)
        graphs.append((gr, ins, outs, torch.cuda.Stream(), c, ln))  # a graph does not keep what it reads alive
    torch.cuda.synchronize()
    for i in range(steps):
        for gr, ins, _, s, _, _ in graphs:
            with torch.cuda.stream(s):
                for t, x in zip(ins, (k, v, q, logits, u)):
                    t.copy_(x[i])
                gr.replay()
        torch.cuda.synchronize()
        for _, _, outs, *_ in graphs:
            for got, ref in zip(outs, want[i]):
                assert torch.equal(got, ref), i
    _status()


# ---- sampling ----------------------------------------------------------------------
def _rows(M, V, dtype, g, spread=2.0, pad=0):
    x = torch.full((M, V + pad), math.nan, device="cuda")
    x[:, :V] = spread * torch.randn(M, V, device="cuda", generator=g)
    lift = torch.randint(0, V, (M, 20), device="cuda", generator=g)
    x[:, :V].scatter_add_(1, lift, 10 * torch.rand(M, 20, device="cuda", generator=g))
    return x.to(dtype)


def _want(x, V, u, t, k, p, m):
    at = lambda s, i: float(s[i]) if torch.is_tensor(s) else float(s)  # noqa: E731
    return [O.sample_row(x[i, :V], float(u[i]), at(t, i), int(at(k, i)), at(p, i), at(m, i)) for i in range(x.shape[0])]


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.8, 200, 1.0, 0.0), (0.9, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.05), (0.7, 40, 0.95, 0.02),
            (1.0, 1, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (-1.0, 5, 0.5, 0.5), (2.0, 3, 0.3, 0.0), (1.0, 0, 1e-6, 0.0),
            (1.0, 0, 0.999999, 0.0), (1e-3, 0, 0.9, 0.0), (50.0, 0, 0.7, 0.0), (1.0, 10 ** 9, 2.0, -1.0), (1.0, 0, 0.0, 0.0),
            (1.0, 0, 1.0, 1.0), (1.0, 0, 1.0, 1.5), (math.inf, 7, 1.0, 0.0), (1.0, -3, 0.5, 0.0)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("V,pad", [(1, 0), (2, 6), (31, 1), (1000, 24), (4097, 0), (50257, 47)])
def test_sampling_of_every_setting(V, pad, dtype):
    K, g = _k(), _gen(V)
    x = _rows(6, V, dtype, g, pad=pad)
    u = torch.rand(6, device="cuda", generator=g)
    u[0], u[1] = 0.0, 1 - 2.0 ** -24
    for t, k, p, m in SETTINGS:
        got = K.sample_tokens(x, V, u, temperature=t, top_k=k, top_p=p, min_p=m)
        assert got.tolist() == _want(x, V, u, t, k, p, m), (t, k, p, m)
    _status()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sampling_with_settings_of_each_row(dtype):
    K, g = _k(), _gen(2)
    n = len(SETTINGS)
    x = _rows(n, 5003, dtype, g)
    u = torch.rand(n, device="cuda", generator=g)
    t, p, m = (torch.tensor([s[i] for s in SETTINGS], device="cuda") for i in (0, 2, 3))
    k = torch.tensor([s[1] for s in SETTINGS], device="cuda")
    got = K.sample_tokens(x, 5003, u, temperature=t, top_k=k, top_p=p, min_p=m)
    assert got.tolist() == _want(x, 5003, u, t, k, p, m)
    for i in range(n):  # a row's token is its own, whatever the others are
        one = K.sample_tokens(x[i:i + 1], 5003, u[i:i + 1], temperature=t[i:i + 1], top_k=k[i:i + 1], top_p=float(p[i]),
                              min_p=m[i:i + 1])
        assert one.tolist() == [int(got[i])]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_sampling_of_equal_logits(dtype):
    """Equal logits go by index: at the largest, at the cut of top-k and inside the nucleus. Borders fall on whole numbers."""
    K = _k()
    x = torch.zeros(8, 1000, device="cuda", dtype=dtype)
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.999, 0.125, 0.3, 1 - 2.0 ** -24], device="cuda")
    for t, k, p, m in [(1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 10, 1.0, 0.0), (1.0, 0, 0.5, 0.0), (1.0, 100, 0.25, 0.5)]:
        assert K.sample_tokens(x, 1000, u, t, k, p, m).tolist() == _want(x, 1000, u, t, k, p, m), (t, k, p, m)
    x[:, ::3] = 2.0
    x[:, 1::3] = -0.0
    for t, k, p, m in [(1.0, 400, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (0.5, 0, 0.97, 0.0), (1.0, 500, 0.9, 0.0), (1.0, 334, 0.5, 0.1),
                       (1.0, 0, 0.5, 0.0)]:
        assert K.sample_tokens(x, 1000, u, t, k, p, m).tolist() == _want(x, 1000, u, t, k, p, m), (t, k, p, m)


def test_sampling_of_masked_and_broken_rows():
    """-inf and the type's lowest value as masks, rows with nothing left, infinities, NaN, and settings that are none."""
    K, g = _k(), _gen(7)
    for dtype in (BF16, F16, F32):
        x = _rows(10, 3001, dtype, g)
        x[0] = -math.inf
        x[1, 1:] = -math.inf
        x[2, torch.randperm(3001, device="cuda", generator=g)[:2990]] = -math.inf
        x[3, 77] = math.nan
        x[4, 5] = math.inf
        x[5] = torch.finfo(dtype).min
        x[6, 100:] = torch.finfo(dtype).min
        x[7] = torch.finfo(dtype).max
        x[8] = -math.inf
        x[8, 3000] = torch.finfo(dtype).min
        x[9] += 1000
        u = torch.rand(10, device="cuda", generator=g)
        for s in [(1.0, 0, 1.0, 0.0), (0.7, 20, 0.9, 0.0), (0.0, 0, 1.0, 0.0), (1.0, 0, 0.99, 0.01), (math.inf, 0, 0.5, 0.0), (math.inf, 9, 1.0, 1.0)]:
            assert K.sample_tokens(x, 3001, u, *s).tolist() == _want(x, 3001, u, *s), s
        assert K.sample_tokens(x, 3001, u)[[0, 3, 4]].tolist() == [-1, -1, -1]
    bad = torch.full((10,), math.nan, device="cuda")
    for s in (dict(temperature=bad), dict(top_p=bad), dict(min_p=bad)):
        assert K.sample_tokens(x, 3001, u, **s).tolist() == [-1] * 10
    assert K.sample_tokens(x, 3001, bad).tolist() == [-1] * 10
    out = torch.tensor([-1.0, 1.0, 2.0, math.inf, -math.inf, 0.0, 1.0, 0.0, 0.0, 1.0], device="cuda")  # clamped to [0, 1)
    assert K.sample_tokens(x, 3001, out).tolist() == _want(x, 3001, out.clamp(0, 1 - 2.0 ** -30), 1.0, 0, 1.0, 0.0)
    _status()


def test_sampling_strides_and_sizes():
    K, g = _k(), _gen(12)
    buf = _rows(40, 9000, BF16, g)
    u = torch.rand(40, device="cuda", generator=g)
    for first, V in ((0, 9000), (1, 4000), (3, 2047), (8, 8192), (5, 1)):
        x = buf[::2, first:first + V]
        assert K.sample_tokens(x, V, u[:20].contiguous(), 0.8, 30, 0.9).tolist() == _want(x, V, u, 0.8, 30, 0.9, 0.0), (first, V)
    one = buf[3:4].expand(40, 9000)
    assert K.sample_tokens(one, 9000, u, 1.1).tolist() == _want(one, 9000, u, 1.1, 0, 1.0, 0.0)
    assert K.sample_tokens(buf[:0], 9000, u[:0]).shape == (0,)
    wide = _rows(3, 2 ** 19, BF16, g)
    for s in ((1.0, 0, 1.0, 0.0), (0.9, 1000, 0.99, 0.0), (3.0, 0, 0.9, 0.0)):
        assert K.sample_tokens(wide, 2 ** 19, u[:3], *s).tolist() == _want(wide, 2 ** 19, u, *s)
    many = _rows(700, 517, F32, g)
    uu = torch.rand(700, device="cuda", generator=g)
    assert K.sample_tokens(many, 517, uu, 0.9, 0, 0.8).tolist() == _want(many, 517, uu, 0.9, 0, 0.8, 0.0)


@pytest.mark.parametrize("dtype,V", [(BF16, 60000), (F32, 60000), (F16, 130001), (F32, 130001), (BF16, 300000)])
def test_sampling_where_nothing_short_holds_what_is_kept(dtype, V):
    """Flat logits, cuts far down, ties without end: more candidates than a list has, rows that shared memory does not hold."""
    K, g = _k(), _gen(V)
    x = _rows(4, V, dtype, g, spread=1.0)
    x[1] = 0.5
    x[2] = (x[2] * 4).round() / 4  # few different values
    x[3, ::2] = -math.inf
    u = torch.rand(4, device="cuda", generator=g)
    for s in [(1.0, 0, 1.0, 0.0), (1.0, 900, 1.0, 0.0), (1.3, 5000, 0.7, 0.0), (1.0, V - 1, 0.999, 0.0), (2.0, 0, 0.99, 0.0),
              (1.5, 0, 0.5, 0.0), (1.0, 0, 0.99999, 0.0), (1.0, 0, 1.0, 1e-7), (0.6, 0, 0.9, 1e-4), (3.0, 3000, 0.95, 0.001)]:
        assert K.sample_tokens(x, V, u, *s).tolist() == _want(x, V, u, *s), s
    _status()


def test_sampling_many_rows_of_unlike_settings():
    """More rows than the GPU has SMs, each of its own kind."""
    K, g = _k(), _gen(21)
    M, V = 400, 20011
    x = _rows(M, V, BF16, g)
    x[::7] *= 0.3
    u = torch.rand(M, device="cuda", generator=g)
    r = torch.rand(4, M, device="cuda", generator=g)
    t = torch.where(r[0] < 0.1, 0.0, 0.2 + 1.5 * r[0])
    k = torch.where(r[1] < 0.4, 0, (800 * r[1]).long())
    p = torch.where(r[2] < 0.3, 1.0, r[2])
    m = torch.where(r[3] < 0.6, 0.0, 0.1 * r[3])
    got = K.sample_tokens(x, V, u, t, k, p, m)
    assert got.tolist() == _want(x, V, u, t, k, p, m)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_sampling_at_the_ends_of_the_range(dtype):
    """Logits and temperatures from the smallest to the largest numbers: all in one row, and next to masks of either kind."""
    K, g = _k(), _gen(31)
    top = torch.finfo(dtype).max
    x = _rows(8, 2003, dtype, g)
    x[1], x[2], x[3] = x[1] * 1e-30, x[2] * (top / 64), x[3] * 1e-38
    x[4] = -top
    x[4, ::7], x[4, 5::7] = -math.inf, -top * 0.99
    x[5, ::2], x[5, 1::4] = top, -top
    x[6] = 0.0
    x[6, 3::5], x[6, 4::5] = -torch.finfo(dtype).tiny, -math.inf
    x[7, 1:] = -math.inf
    u = torch.rand(8, device="cuda", generator=g)
    for t in (1e-40, 1e-30, 1e-7, 1e5, 1e30, 2.0 ** 121, 3e38, 1e300, math.inf):
        for k, p, m in ((0, 1.0, 0.0), (9, 1.0, 0.0), (0, 0.6, 0.0), (50, 0.9, 0.1)):
            assert K.sample_tokens(x, 2003, u, t, k, p, m).tolist() == _want(x, 2003, u, t, k, p, m), (t, k, p, m)
    _status()


def test_sampling_follows_the_distribution():
    """Numbers spread evenly over [0, 1) give every token its share: each border is at its running probability."""
    K, g = _k(), _gen(13)
    x = (3 * torch.randn(1, 50, device="cuda", generator=g)).to(F32)
    n = 4096
    u = (torch.arange(n, device="cuda") + 0.5) / n
    got = torch.bincount(K.sample_tokens(x.expand(n, 50), 50, u, 0.7), minlength=50)
    p = torch.softmax(x[0].double() / 0.7, 0)
    assert bool((got.double() - n * p).abs().max() <= 1)
