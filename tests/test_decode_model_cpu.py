"""Generation on the fused engine (models/decode.py) with the kernels emulated: the host code around them, and the cuts of the
plain sampler."""
import pytest
import torch

import decode_oracle as O
from decode_emulation import emulate

from heiretsu_b200.config import GPTConfig
from heiretsu_b200.models.decode import Decoder
from heiretsu_b200.models.generate import _pick, generate
from heiretsu_b200.models.gpt import GPT

CFG = dict(block_size=64, vocab_size=200, n_layer=3, n_head=2, n_embed=128)


def _model(dtype=torch.float32, moe=False, seed=0):
    from heiretsu_b200.parallel.flat import FlatParams

    torch.manual_seed(seed)
    m = GPT(GPTConfig(**CFG, **(dict(num_experts=4, top_k=2, moe_freq=2) if moe else {})))
    with torch.no_grad():  # scores that are not all alike
        for blk in m.tr.h:
            blk.attn.c_attn.weight.mul_(6)
    FlatParams(m, torch.device("cpu"), dtype16=dtype)
    return m


def _ids(b, n, seed=1):
    return torch.randint(0, 200, (b, n), generator=torch.Generator().manual_seed(seed))


def test_greedy_tokens_are_those_of_the_plain_model(monkeypatch):
    """With stand-ins in 32 bits every step's logits are the whole model's."""
    emulate(monkeypatch)
    m = _model()
    idx = _ids(3, 7)
    want = generate(m, idx, 40, temperature=0)
    d = Decoder(m, 3, page_size=16)
    logits = d.append(idx)
    with torch.no_grad():
        assert torch.allclose(logits, m(idx)[0][:, -1], atol=1e-4)
    first, second = d.generate(15, temperature=0), d.generate(25, temperature=0)
    assert torch.equal(torch.cat([idx, first, second], 1), want)
    assert d.lens == [46] * 3 and d.lengths.tolist() == d.lens
    got = generate(m, idx, 40, temperature=0, engine="fused")
    assert torch.equal(got, want) and m.training


def test_prompts_of_unlike_lengths_and_what_is_added_later(monkeypatch):
    emulate(monkeypatch)
    m = _model()
    idx, more = _ids(3, 9), _ids(3, 11, seed=4)
    n1, n2 = [9, 1, 4], [2, 11, 5]
    d = Decoder(m, 3, page_size=16)
    d.append(idx, n1)
    a = d.generate(6, temperature=0)
    d.append(more, n2)
    b = d.generate(10, temperature=0)
    for i in range(3):
        x = idx[i:i + 1, : n1[i]]
        w1 = generate(m, x, 6, temperature=0)
        assert torch.equal(w1[0, -6:], a[i])
        w2 = generate(m, torch.cat([w1, more[i:i + 1, : n2[i]]], 1), 10, temperature=0)
        assert torch.equal(w2[0, -10:], b[i]), i
    assert d.lens == [n1[i] + n2[i] + 6 + 9 for i in range(3)]


@pytest.mark.parametrize("steps", [1, 4])
def test_a_call_that_fails_can_be_made_again(monkeypatch, steps):
    """An error in the middle of append or generate (memory that runs out, say) leaves the sequences as they were."""
    from heiretsu_b200.models import decode

    emulate(monkeypatch)
    m = _model()
    idx = _ids(2, 5)
    want = generate(m, idx, 12, temperature=0)
    d = Decoder(m, 2, page_size=16)
    calls = []

    def failing(name, at):
        real = getattr(decode.K, name)

        def call(*a, **kw):
            calls.append(name)
            if len(calls) == at:
                raise RuntimeError("out of memory")
            return real(*a, **kw)

        calls.clear()
        monkeypatch.setattr(decode.K, name, call)
        return lambda: monkeypatch.setattr(decode.K, name, real)

    for prompt in (idx[:, :3], idx[:, 3:]):
        undo = failing("kv_write", 2)
        with pytest.raises(RuntimeError, match="out of memory"):
            d.append(prompt)
        undo()
        d.append(prompt)
    out = []
    for _ in range(2):
        undo = failing("sample_tokens", steps)
        with pytest.raises(RuntimeError, match="out of memory"):
            d.generate(6, temperature=0)
        undo()
        assert d.lengths.tolist() == d.lens and m.training
        out.append(d.generate(6, temperature=0))
    assert torch.equal(torch.cat([idx, *out], 1), want)


def test_mixture_of_experts_and_8_bits(monkeypatch):
    from moe_emulation import emulate_moe

    emulate(monkeypatch)
    emulate_moe(monkeypatch.setattr)
    m = _model(torch.bfloat16, moe=True)
    out = generate(m, _ids(2, 5), 12, temperature=0, engine="fused", cache_bits=8)
    assert out.shape == (2, 17)
    m = _model()
    idx = _ids(4, 30)
    d16, d8 = Decoder(m, 4), Decoder(m, 4, cache_bits=8)
    a, b = d16.append(idx), d8.append(idx)
    assert torch.equal(a, b)  # a first prompt's attention runs on what is not yet quantised
    with torch.no_grad():
        x, y = d16._step(idx[:, 0]), d8._step(idx[:, 0])
    off = (x - y).norm() / x.norm()
    assert 0 < off < 0.02, off  # values off by 1/254 of their head's largest on average


def test_sampled_tokens_follow_the_settings(monkeypatch):
    emulate(monkeypatch)
    m = _model()
    idx = _ids(2, 4)
    s = dict(temperature=0.7, top_k=20, top_p=0.9, min_p=0.05)
    d = Decoder(m, 2)
    logits = d.append(idx)
    got = d.generate(8, generator=torch.Generator().manual_seed(3), **s)
    u = torch.rand(8, 2, generator=torch.Generator().manual_seed(3))
    for i in range(8):
        assert got[:, i].tolist() == [O.sample_row(logits[b], float(u[i, b]), s["temperature"], 20, 0.9, 0.05) for b in range(2)]
        idx = torch.cat([idx, got[:, i:i + 1]], 1)
        with torch.no_grad():
            logits = m(idx)[0][:, -1]


def test_pages_are_shared_and_run_out(monkeypatch):
    emulate(monkeypatch)
    m = _model()
    d = Decoder(m, 2, page_size=16, pages=5)
    d.append(_ids(2, 40), [40, 3])  # 3 pages and 1
    assert len(d.free) == 1
    before = (d.lens[:], [o[:] for o in d.owned])
    with pytest.raises(ValueError, match="free pages"):
        d.append(_ids(2, 20), [10, 20])
    assert (d.lens, d.owned) == before
    d.append(_ids(2, 14), [1, 14])  # the last one
    assert len(d.free) == 0 and len({p for o in d.owned for p in o}) == 5


def test_refusals(monkeypatch):
    emulate(monkeypatch)
    m = _model()
    with pytest.raises(ValueError, match="block_size"):
        generate(m, _ids(1, 30), 40, engine="fused")
    with pytest.raises(ValueError, match="from a cache"):
        generate(m, _ids(1, 3), 4, engine="fused", kv_cache=False)
    with pytest.raises(ValueError, match="plain or fused"):
        generate(m, _ids(1, 3), 4, engine="other")
    with pytest.raises(ValueError, match="8 bits"):
        generate(m, _ids(1, 3), 4, cache_bits=8)
    with pytest.raises(ValueError, match="16 or 8 bits"):
        Decoder(m, 1, cache_bits=4)
    with pytest.raises(ValueError, match="at least one"):
        Decoder(m, 0)
    with pytest.raises(ValueError, match="FlatParams"):
        Decoder(GPT(GPTConfig(**CFG)), 1)
    d = Decoder(m, 2)
    with pytest.raises(ValueError, match="append a prompt"):
        d.generate(3)
    for idx, n in ((_ids(1, 3), None), (_ids(2, 0), None), (_ids(2, 3), [0, 3]), (_ids(2, 3), [4, 3]), (_ids(2, 3), [3])):
        with pytest.raises(ValueError):
            d.append(idx, n)
    d.append(_ids(2, 60))
    with pytest.raises(ValueError, match="block_size"):
        d.generate(6)
    assert d.generate(4, temperature=0).shape == (2, 4) and d.generate(0).shape == (2, 0)
    with pytest.raises(ValueError, match="block_size"):
        d.generate(1)


@pytest.mark.parametrize("top_k,top_p,min_p", [(None, 0.6, 0.0), (None, 1.0, 0.2), (5, 0.9, 0.1), (None, 1e-9, 0.0), (None, 1.0, 1.0)])
def test_plain_sampler_cuts(top_k, top_p, min_p):
    """Tokens drawn by the plain sampler are those that the definition keeps, at their shares."""
    g = torch.Generator().manual_seed(0)
    x = 2 * torch.randn(1, 40, generator=g)
    n = 20000
    got = torch.bincount(_pick(x.expand(n, 40), 0.8, top_k, g, top_p, min_p)[:, 0], minlength=40).double()
    y, order = (x[0].double() / 0.8).sort(descending=True, stable=True)
    p = torch.softmax(y, 0)
    if top_k:
        p[top_k:] = 0
        p = p / p.sum()
    keep = (p.cumsum(0) - p < top_p) & (p >= min_p * p[0])
    keep[0] = True
    p = torch.where(keep, p, 0.0)
    want = torch.zeros(40, dtype=torch.float64).scatter_(0, order, n * p / p.sum())
    assert bool((got[want == 0] == 0).all())
    # a share of n draws has a standard deviation of sqrt(n p (1 - p)): 6 of them
    assert bool(((got - want).abs() <= 6 * torch.sqrt(want * (1 - want / n)) + 1e-6).all())


def test_model_method_takes_the_plain_path_on_a_cpu():
    m = GPT(GPTConfig(**CFG))
    idx = _ids(1, 3)
    assert torch.equal(m.generate(idx, 5, temperature=0), generate(m, idx, 5, temperature=0))
