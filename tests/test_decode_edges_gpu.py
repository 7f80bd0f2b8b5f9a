"""Calls of the decoder and of the decoding operators that are easy to get wrong, on a GPU."""
import pytest
import torch

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
