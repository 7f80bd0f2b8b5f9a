"""Generation on the fused engine (models/decode.py) on a GPU: the kernels together, as a decoder uses them."""
import os
import subprocess
import sys
from dataclasses import asdict

import pytest
import torch

from heiretsu_b200.config import GPTConfig

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _model(dtype=torch.bfloat16, moe=False, heads=4, width=256, vocab=1000):
    from heiretsu_b200.models.gpt import GPT
    from heiretsu_b200.parallel.flat import FlatParams

    torch.manual_seed(0)
    kw = dict(num_experts=4, top_k=2, moe_freq=2) if moe else {}
    m = GPT(GPTConfig(block_size=256, vocab_size=vocab, n_layer=3, n_head=heads, n_embed=width, dropout=0.0, **kw)).cuda()
    with torch.no_grad():
        for blk in m.tr.h:
            blk.attn.c_attn.weight.mul_(4)
    FlatParams(m, torch.device("cuda"), dtype16=dtype)
    m.fused = True
    return m.eval()


def _ids(b, n, vocab=1000, seed=1):
    return torch.randint(0, vocab, (b, n), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def _status():
    from heiretsu_b200.ops._C import check_status
    check_status(torch.cuda.current_device())


@pytest.mark.parametrize("dtype,heads,width", [(torch.bfloat16, 4, 256), (torch.float16, 2, 256), (torch.bfloat16, 8, 256), (torch.bfloat16, 8, 128)])
def test_steps_give_the_whole_forwards_logits(dtype, heads, width):
    """Prompt, single tokens and tokens added later against the fused forward over the whole sequence. Both round the same
    operands to 16 bits; the orders of their sums differ, so single roundings do: the difference is bounded by that of
    the fused forward to the plain fp32 model, which rounds nothing."""
    from heiretsu_b200.models.decode import Decoder

    m = _model(dtype, heads=heads, width=width)
    idx = _ids(3, 200)
    with torch.no_grad():
        full = m(idx)[0].float()
        m.fused = False
        plain = m(idx)[0].float()
        m.fused = True
    noise = (full - plain).norm() / plain.norm()
    d = Decoder(m, 3, page_size=16)
    close = lambda a, t: float((a.float() - full[:, t]).norm() / full[:, t].norm())  # noqa: E731
    assert close(d.append(idx[:, :100]), 99) <= noise
    d._reserve([20] * 3)
    for t in range(100, 120):
        with torch.no_grad():
            off = close(d._step(idx[:, t])[:, :1000], t)
        assert off <= 1.5 * noise, (t, off, float(noise))
    d.lens = [120] * 3
    assert close(d.append(idx[:, 120:200]), 199) <= 1.5 * noise
    _status()


def test_unlike_lengths_match_each_sequence_alone():
    from heiretsu_b200.models.decode import Decoder

    m = _model()
    idx = _ids(4, 90)
    n = [90, 1, 33, 64]
    d = Decoder(m, 4, page_size=32)
    logits = d.append(idx, n)
    with torch.no_grad():
        for b in range(4):
            want = m(idx[b:b + 1, : n[b]])[0][0, -1].float()
            assert (logits[b].float() - want).norm() <= 0.02 * want.norm()
    d.generate(12, temperature=0)
    assert d.lengths.tolist() == [x + 11 for x in n]
    _status()


@pytest.mark.parametrize("bits,moe", [(16, False), (8, False), (16, True)])
def test_graphs_give_the_tokens_of_single_steps(bits, moe):
    from heiretsu_b200.models.decode import Decoder

    m = _model(moe=moe)
    idx = _ids(5, 20)
    out = []
    for graph in (True, False):
        d = Decoder(m, 5, cache_bits=bits)
        g = torch.Generator(device="cuda").manual_seed(5)
        d.append(idx)
        a = d.generate(40, temperature=0.9, top_k=50, top_p=0.95, min_p=0.01, generator=g, cuda_graph=graph)
        b = d.generate(30, temperature=0, generator=g, cuda_graph=graph)
        d.append(idx)
        c = d.generate(25, temperature=1.1, generator=g, cuda_graph=graph)
        out.append(torch.cat([a, b, c], 1))
    assert torch.equal(out[0], out[1])
    assert bool(((out[0] >= 0) & (out[0] < 1000)).all())
    _status()


def test_8_bits_stay_near_16():
    from heiretsu_b200.models.decode import Decoder

    m = _model()
    idx = _ids(4, 150)
    a, b = Decoder(m, 4), Decoder(m, 4, cache_bits=8)
    a.append(idx), b.append(idx)
    with torch.no_grad():
        x, y = a._step(idx[:, 0]).float(), b._step(idx[:, 0]).float()
    assert (x - y).norm() <= 0.03 * x.norm()
    mem = lambda d: sum(t.numel() * t.element_size() for p in d.pools for t in p.values() if t is not None)  # noqa: E731
    assert mem(b) * 1.9 < mem(a)


def test_sampled_tokens_train_a_policy():
    """Samples of the decoder scored by token_logprobs and used by policy_loss: at fresh samples the ratios are 1."""
    m = _model()
    idx = _ids(2, 16)
    out = m.generate(idx, 24, temperature=1.0, generator=torch.Generator(device="cuda").manual_seed(1))
    assert out.shape == (2, 40) and torch.equal(out[:, :16], idx)
    x, y = out[:, :-1].contiguous(), out[:, 1:].clone()
    y[:, :15] = -100
    m.train()
    with torch.no_grad():
        logp = m.token_logprobs(x, y)
    assert bool((logp[:, 15:] < 0).all()) and bool((logp[:, :15] == 0).all())
    loss, aux, _, _ = m.policy_loss(x, y, logp, torch.ones(2, device="cuda"))
    (loss + aux).backward()
    assert abs(float(loss.detach()) + 1) < 1e-5  # -(mean of ratio 1 times advantage 1)


def test_model_method_without_a_cache():
    m = _model()
    idx = _ids(2, 6)
    out = m.generate(idx, 5, temperature=0, kv_cache=False)
    assert torch.equal(out, m.generate(idx, 5, temperature=0, engine="plain"))


def test_sample_script_on_the_fused_engine(tmp_path):
    m = _model(vocab=300)
    torch.save({"model": m.state_dict(), "cfg": asdict(m.cfg), "step": 1}, tmp_path / "dense.pt")
    lines = []
    for extra in (["--cache_bits", "16"], ["--cache_bits", "8", "--top_p", "0.9", "--min_p", "0.01"]):
        r = subprocess.run([sys.executable, os.path.join(ROOT, "sample.py"), "--ckpt", str(tmp_path / "dense.pt"), "--start", "1,2,3",
                            "--max_new_tokens", "20", "--num_samples", "3", "--engine", "fused", *extra], capture_output=True,
                           text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]
        rows = [[int(t) for t in line.split(",")] for line in r.stdout.strip().splitlines()[:3]]
        assert all(len(row) == 23 and row[:3] == [1, 2, 3] and max(row) < 300 for row in rows)
        lines.append(rows)
    assert lines[0] != lines[1]
