"""Calls of the decoder and of the decoding operators that are easy to get wrong, on a GPU."""
import pytest
import torch

import test_decode_gpu as T

from heiretsu_b200.config import GPTConfig

pytestmark = pytest.mark.gpu


def _model(dtype=torch.bfloat16, moe=False, heads=4, width=256, vocab=1000, device="cuda"):
    from heiretsu_b200.models.gpt import GPT
    from heiretsu_b200.parallel.flat import FlatParams

    torch.manual_seed(0)
    kw = dict(num_experts=4, top_k=2, moe_freq=2) if moe else {}
    m = GPT(GPTConfig(block_size=256, vocab_size=vocab, n_layer=3, n_head=heads, n_embed=width, dropout=0.0, **kw)).to(device)
    with torch.no_grad():
        for blk in m.tr.h:
            blk.attn.c_attn.weight.mul_(4)
    FlatParams(m, torch.device(device), dtype16=dtype)
    m.fused = True
    return m.eval()


def _ids(b, n, vocab=1000, seed=1):
    return torch.randint(0, vocab, (b, n), generator=torch.Generator().manual_seed(seed)).cuda()


def _status():
    from heiretsu_b200.ops._C import check_status
    check_status(torch.cuda.current_device())


@pytest.mark.parametrize("first", [False, True])
def test_a_model_on_the_device_that_is_not_current(first):
    """A graph gives the tokens of single steps, whether the process has captured on the current device before or not."""
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    from heiretsu_b200.models.decode import Decoder

    if first:
        Decoder(_model(), 1).append(_ids(1, 3))
        x, g = torch.zeros(4, device="cuda:0"), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x += 1
    m = _model(device="cuda:1")
    out = []
    for graph in (True, False):
        d = Decoder(m, 3)
        d.append(_ids(3, 9))
        out.append(d.generate(30, temperature=0, cuda_graph=graph))
        assert d.lengths.tolist() == d.lens and torch.cuda.current_device() == 0
    assert torch.equal(*out)


def test_captures_between_other_captures():
    """A decoder's graph neither takes nor leaves anything of another graph's, and the current stream may be any."""
    from heiretsu_b200.models.decode import Decoder

    m, idx = _model(), _ids(3, 9)
    x, g = torch.zeros(4, device="cuda"), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x += 1
    out = []
    for graph in (True, False):
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            d = Decoder(m, 3)
            d.append(idx)
            out.append(d.generate(30, temperature=0, cuda_graph=graph))
            g.replay()
        torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(*out) and x.tolist() == [2.0] * 4
    _status()


@pytest.mark.parametrize("moe", [False, True])
def test_tokens_behind_a_sequences_own_may_be_anything(moe):
    """Padding that is no token of the vocabulary changes nothing, in a first prompt and in tokens added later, and is no error."""
    from heiretsu_b200.models.decode import Decoder

    m, out = _model(moe=moe), []
    for fill in (0, -100):
        d, logits = Decoder(m, 3), []
        for seed, n in ((1, [90, 1, 37]), (2, [2, 41, 33])):
            idx = _ids(3, 90, seed=seed)
            for b in range(3):
                idx[b, n[b]:] = fill
            logits.append(d.append(idx, n))
        out.append((*logits, d.generate(12, temperature=0)))
    assert all(torch.equal(a, b) for a, b in zip(*out))
    _status()


@pytest.mark.parametrize("moe,graph", [(False, True), (True, True), (True, False)])
def test_a_row_without_a_token_is_an_error(moe, graph):
    """One sequence's cache holds NaN: generate says so, leaves all as they were and no error behind; the cache mended, it gives what it
    would have given."""
    from heiretsu_b200.models.decode import Decoder

    m = _model(moe=moe)
    d, ref = Decoder(m, 3), Decoder(m, 3)
    for x in (d, ref):
        x.append(_ids(3, 30))
    want = torch.cat([ref.generate(n, temperature=0, cuda_graph=graph) for n in (6, 25)], 1)
    assert torch.equal(d.generate(6, temperature=0, cuda_graph=graph), want[:, :6])
    pool, page = d.pools[1]["v_pages"], d.owned[1][0]
    kept = pool[page].clone()
    pool[page, 2, 7, 5] = float("nan")
    with pytest.raises(RuntimeError, match=r"no token for sequences \[1\]"):
        d.generate(25, temperature=0, cuda_graph=graph)
    _status()
    assert d.lens == [35] * 3 and d.lengths.tolist() == d.lens
    pool[page] = kept
    assert torch.equal(d.generate(25, temperature=0, cuda_graph=graph), want[:, 6:])
    _status()


# ---- what generate gives, against the whole forward ----------------------------------
@pytest.mark.parametrize("bits", [16, 8])
def test_greedy_tokens_are_the_whole_forwards(bits):
    """Tokens of generate, generate again, append and generate, checked one by one against the fused forward over all of them:
    a token's logit is the row's largest but for what the two may differ by.

    E is the largest distance of a fused logit to the plain fp32 model's. The decoder rounds the same operands in other orders
    of summation: its logits are within 2 E of the plain ones. It takes c where its logit of c is no less than that of the row's
    largest, so in the fused forward c is behind by at most 2 (2 E + E). In 8 bits K and V are off by up to 1/127 of
    their head's largest, instead of 2^-8 of themselves: with a largest of 2.5 root mean squares, 5 times as far, which
    makes 2 (1 + 5) E of the 2 E."""
    from heiretsu_b200.models.decode import Decoder

    m, idx, more = _model(), _ids(4, 21), _ids(4, 17, seed=7)
    d = Decoder(m, 4, cache_bits=bits, page_size=16)
    d.append(idx)
    a, b = d.generate(30, temperature=0), d.generate(12, temperature=0)
    d.append(more)
    c = d.generate(40, temperature=0)
    _status()
    whole = torch.cat([idx, a, b, more, c], 1)
    with torch.no_grad():
        full = m(whole)[0].float()
        m.fused = False
        plain = m(whole)[0].float()
    E = (full - plain).abs().max()
    behind = full[:, :-1].amax(-1) - full[:, :-1].gather(2, whole[:, 1:, None])[..., 0]
    own = torch.ones_like(behind, dtype=torch.bool)
    own[:, :20] = own[:, 62:79] = False  # the prompts
    assert float(behind[own].max()) <= (2 * (2 + 1) if bits == 16 else 2 * (12 + 1)) * float(E)
    assert float(behind[~own].median()) > 30 * float(E)  # other tokens are far behind
    assert int(own.sum()) == 4 * 82


@pytest.mark.parametrize("bits,graph", [(16, True), (8, True), (16, False)])
def test_sampled_tokens_are_those_of_single_calls(bits, graph):
    """Each step's token is that of sample_tokens on its logits with its row of the uniform numbers, from call to call."""
    from heiretsu_b200.models.decode import Decoder
    from heiretsu_b200.ops import kernels as K

    m, idx = _model(), _ids(5, 19)
    s = dict(temperature=0.9, top_k=80, top_p=0.95, min_p=0.001)
    d, ref = Decoder(m, 5, cache_bits=bits), Decoder(m, 5, cache_bits=bits)
    d.append(idx)
    g = torch.Generator(device="cuda").manual_seed(9)
    got = torch.cat([d.generate(n, generator=g, cuda_graph=graph, **s) for n in (25, 1, 14)], 1)
    g = torch.Generator(device="cuda").manual_seed(9)
    u = torch.cat([torch.rand(n, 5, device="cuda", generator=g) for n in (25, 1, 14)])
    logits = ref.append(idx)
    ref._reserve([39] * 5)
    with torch.no_grad():
        for t in range(40):
            token = K.sample_tokens(logits, 1000, u[t], **s)
            assert torch.equal(token, got[:, t]), t
            if t < 39:
                logits = ref._step(token)
    _status()


# ---- caches of other layouts -----------------------------------------------------------
LAYOUTS = {  # memory of [pages, heads, slots, channels]: dimensions from the outermost, and channels between slots
    "slots, heads": ((0, 2, 1, 3), 0), "heads, slots apart": ((0, 1, 2, 3), 16), "heads outermost": ((1, 0, 2, 3), 0),
    "slots, heads apart": ((0, 2, 1, 3), 32), "slots outermost": ((2, 0, 1, 3), 0),
}


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 8), (torch.float16, 8), (torch.bfloat16, 16), (torch.float16, 16)])
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 16), (6, 2, 32), (5, 5, 64), (8, 4, 128)])
def test_attention_over_caches_of_other_layouts(heads, kv, dim, dtype, bits, layout):
    """Slots that do not follow one another, at every length of a token (16 to 256 bytes), pages that hold whole tiles and
    pages that do not: what the packed cache gives, bit by bit, and within the bounds of the definition."""
    from heiretsu_b200.ops import kernels as K

    order, gap = LAYOUTS[layout]
    lengths = [1, 0, 16, 63, 130, 259, 513]
    for size in (16, 48, 64):
        q, c, table, n, held = T._batch(lengths, heads, kv, dim, size, dtype, bits, seed=heads + dim + size)
        want, want_lse = K.decode_attention(q, table=table, lengths=n, **c.pools)
        pools = dict(c.pools)
        for name in ("k_pages", "v_pages"):
            x = c.pools[name]
            sizes = [x.shape[i] for i in order]
            sizes[-1] += gap
            mem = torch.full(sizes, 3, device="cuda", dtype=x.dtype)[..., :dim]
            pools[name] = mem.permute([order.index(i) for i in range(4)])
            pools[name].copy_(x)
        out, lse = K.decode_attention(q, table=table, lengths=n, **pools)
        T._compare(out, lse, q, held)
        assert torch.equal(out, want) and torch.equal(lse, want_lse), size
    _status()
