"""Calls of the decoder and of the decoding operators that are easy to get wrong: other devices, padded batches, broken rows,
settings at their ends. The host code, on emulated kernels (``decode_emulation``)."""
import contextlib
import itertools
from types import SimpleNamespace

import pytest
import torch

from decode_emulation import emulate

from heiretsu_b200.config import GPTConfig
from heiretsu_b200.models import decode
from heiretsu_b200.models.decode import Decoder
from heiretsu_b200.models.gpt import GPT
from heiretsu_b200.ops import _C
from heiretsu_b200.ops import kernels as K

CFG = dict(block_size=64, vocab_size=200, n_layer=2, n_head=2, n_embed=128)


def _model(seed=0, **kw):
    from heiretsu_b200.parallel.flat import FlatParams

    torch.manual_seed(seed)
    m = GPT(GPTConfig(**CFG), **kw)
    FlatParams(m, torch.device("cpu"), dtype16=torch.float32)
    return m


def _ids(b, n, seed=1):
    return torch.randint(0, 200, (b, n), generator=torch.Generator().manual_seed(seed))


class FakeCuda:
    """As much of ``torch.cuda`` as generation uses, with device 0 current; notes the device of every capture, replay and wait."""

    def __init__(self):
        self.current, self.seen = 0, []
        fake = self

        class Stream:
            def __init__(self, device=None):
                self.index = fake.current if device is None else torch.device(device).index

            def wait_stream(self, other):
                pass

            def synchronize(self):
                fake.seen.append(("wait", self.index))

        class CUDAGraph:
            def capture_begin(self, *a, **kw):
                fake.seen.append(("capture", fake.current))

            def capture_end(self):
                pass

            def replay(self):
                fake.seen.append(("replay", fake.current))

        self.Stream, self.CUDAGraph = Stream, CUDAGraph
        self.default = Stream()  # where a capture without a stream of its own runs: the device of the first one

    @contextlib.contextmanager
    def device(self, device):
        old, self.current = self.current, torch.device(device).index
        yield
        self.current = old

    @contextlib.contextmanager
    def stream(self, s):
        with self.device(torch.device("cuda", s.index)):
            yield

    @contextlib.contextmanager
    def graph(self, g, stream=None):
        with self.stream(self.default if stream is None else stream):
            g.capture_begin()
            yield
            g.capture_end()

    def current_stream(self, device=None):
        return self.Stream(device)

    def synchronize(self, device=None):
        self.seen.append(("wait", self.Stream(device).index))

    def empty_cache(self):
        pass


def test_a_graph_is_captured_and_replayed_on_the_models_device(monkeypatch):
    """The model is on device 1, device 0 is current: what is captured, replayed and waited for is device 1's."""
    emulate(monkeypatch)
    d = Decoder(_model(), 2, page_size=16)
    d.append(_ids(2, 5))
    fake = FakeCuda()
    here = lambda f: lambda *a, **kw: f(*a, **{k: v for k, v in kw.items() if k != "device"})  # noqa: E731
    torch_ = {n: getattr(torch, n) for n in dir(torch)} | {n: here(getattr(torch, n)) for n in ("rand", "zeros", "tensor")}
    torch_ |= {"cuda": fake, "empty": here(torch.zeros)}
    monkeypatch.setattr(decode, "torch", SimpleNamespace(**torch_))
    d.device = torch.device("cuda", 1)
    d.generate(20, temperature=0)
    assert [w for w, _ in fake.seen].count("capture") == 1 and [w for w, _ in fake.seen].count("replay") == 18
    assert {i for _, i in fake.seen} == {1} and fake.seen[-1][0] == "wait" and fake.current == 0


@pytest.mark.parametrize("pad", [-1, -100, 10 ** 9])
def test_tokens_behind_a_sequences_own_may_be_anything(monkeypatch, pad):
    """Padding that is no token of the vocabulary, in a first prompt and in tokens added later."""
    emulate(monkeypatch)
    m = _model()
    out = []
    for fill in (0, pad):
        d = Decoder(m, 3, page_size=16)
        logits = []
        for seed, n in ((1, [9, 1, 4]), (2, [2, 11, 5])):
            idx = _ids(3, 11, seed)
            for b in range(3):
                idx[b, n[b]:] = fill
            logits.append(d.append(idx, n))
        out.append((logits, d.generate(5, temperature=0)))
    assert all(torch.equal(a, b) for a, b in zip(out[0][0], out[1][0])) and torch.equal(out[0][1], out[1][1])


def test_a_row_without_a_token_is_an_error(monkeypatch):
    """Logits of NaN give no token: generate says which sequence's, and leaves all as they were."""
    emulate(monkeypatch)
    m = _model()
    d, ref = Decoder(m, 3, page_size=16), Decoder(m, 3, page_size=16)
    for x in (d, ref):
        x.append(_ids(3, 5))
    good = d.logits.clone()
    d.logits[1, 3] = float("nan")
    with pytest.raises(RuntimeError, match=r"no token for sequences \[1\]"):
        d.generate(1)
    assert d.lens == [5] * 3 and d.lengths.tolist() == d.lens and m.training
    d.logits = good
    want = ref.generate(9, temperature=0)
    assert torch.equal(d.generate(4, temperature=0), want[:, :4])
    d.pools[0]["k_pages"], kept = torch.full_like(d.pools[0]["k_pages"], float("nan")), d.pools[0]["k_pages"]
    with pytest.raises(RuntimeError, match=r"no token for sequences \[0, 1, 2\]"):
        d.generate(1, temperature=0)
    assert d.lens == [8] * 3 and d.lengths.tolist() == d.lens
    d.pools[0]["k_pages"] = kept
    assert torch.equal(d.generate(5, temperature=0), want[:, 4:])


def test_a_model_that_a_decoder_does_not_take_generates_on_the_plain_modules(monkeypatch):
    """GPT.generate's own choice of engine: the fused one where it has what that needs, and only there."""
    from heiretsu_b200.models import generate as gen

    emulate(monkeypatch)
    engines = []
    monkeypatch.setattr(gen, "generate", lambda model, idx, n, engine="plain", **kw: engines.append(engine))
    idx = SimpleNamespace(is_cuda=True)

    def engine(model, **kw):
        model.fused = True
        engines.clear()
        model.generate(idx, 4, **kw)
        return engines[0]

    assert engine(_model()) == "fused" and engine(_model(), kv_cache=False) == "plain"
    assert engine(_model(), engine="plain") == "plain" and engine(_model(), cache_bits=8) == "fused"
    for topo in (SimpleNamespace(tp=2), SimpleNamespace(ep=2)):
        m = _model()
        m.topo = topo
        assert engine(m) == "plain" and engine(m, engine="fused") == "fused"  # asked for, the decoder refuses
        with pytest.raises(ValueError, match="tp 1 and ep 1"):
            Decoder(m, 1)
    m = GPT(GPTConfig(**CFG))
    assert engine(m) == "plain"
    monkeypatch.setattr(decode, "MAX_VOCAB", 100)
    assert engine(_model()) == "plain"
    with pytest.raises(ValueError, match="vocabulary"):
        Decoder(_model(), 1)
    m = _model()
    m.fused = False
    m.generate(idx, 4)
    assert engines[-1] == "plain"


@pytest.mark.parametrize("top_k", [0, -1, 200, 10 ** 6])
@pytest.mark.parametrize("top_p,min_p", [(1.0, 0.0), (0.6, 0.05)])
def test_a_top_k_of_0_or_of_the_vocabulary_keeps_all(monkeypatch, top_k, top_p, min_p):
    """On either engine; the plain sampler draws what it draws without a top_k."""
    from heiretsu_b200.models.generate import _pick, generate

    x = 3 * torch.randn(64, 200, generator=torch.Generator().manual_seed(2))
    draw = lambda k: _pick(x, 0.8, k, torch.Generator().manual_seed(5), top_p, min_p)  # noqa: E731
    assert torch.equal(draw(top_k), draw(None))
    emulate(monkeypatch)
    m = _model()
    for engine in ("plain", "fused"):
        out = [generate(m, _ids(2, 4), 6, 0.9, k, torch.Generator().manual_seed(3), engine=engine, top_p=top_p, min_p=min_p)
               for k in (top_k, None)]
        assert torch.equal(*out)


needs_extension = pytest.mark.skipif(not _C.available(), reason="the extension is not built")


@needs_extension
def test_writes_to_pools_that_overlap_are_refused():
    """K and V pools that share elements, not only those that begin at one address; pools that lie in each other's gaps are fine."""
    k, slots = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.arange(3)

    def write(match, k_pages, v_pages, **exps):
        with pytest.raises(RuntimeError, match=match):
            K.kv_write(k, k, slots, k_pages, v_pages, **exps)

    buf = torch.zeros(8, 2, 16, 64, dtype=torch.bfloat16)
    write("overlap", buf[:4], buf[3:7])
    write("overlap", buf[3:7], buf[:4])
    write("overlap", buf[::2][:3], buf[4:7])
    write("CUDA", buf[:4], buf[4:])
    write("CUDA", buf[::2], buf[1::2])
    native = torch.zeros(4, 16, 2, 2, 64, dtype=torch.bfloat16)  # [pages, slots, K or V, heads, channels]
    write("CUDA", native[:, :, 0].transpose(1, 2), native[:, :, 1].transpose(1, 2))
    mixed = torch.zeros(4, 2, 2 * 16 * 64, dtype=torch.bfloat16)  # pages of K by heads and V by slots
    write("CUDA", mixed[:, 0].view(4, 2, 16, 64), mixed[:, 1].view(4, 16, 2, 64).transpose(1, 2))
    write("overlap", mixed[:, 0].view(4, 2, 16, 64), mixed[:, 0, 8:].as_strided((4, 2, 16, 64), (4096, 64, 128, 1), 8))
    heads = torch.zeros(4, 5, 16, 64, dtype=torch.bfloat16)
    write("CUDA", heads[:, :2], heads[:, 2:4])
    write("overlap", heads[:, :2], heads[:, 1:3])
    codes, exps = torch.zeros(8, 2, 16, 64, dtype=torch.int8), torch.zeros(8, 2, 16, dtype=torch.uint8)
    write("overlap", codes[:4], codes[4:], k_exp=exps[:4], v_exp=exps[2:6])
    write("overlap", codes[:4], codes[2:6], k_exp=exps[:4], v_exp=exps[4:])
    write("CUDA", codes[:4], codes[4:], k_exp=exps[:4], v_exp=exps[4:])


@needs_extension
def test_what_overlaps_is_what_shares_an_element():
    """Every shift of one small view against another, by listing their elements."""
    k, slots = torch.zeros(1, 2, 16, dtype=torch.bfloat16), torch.arange(1)
    buf = torch.zeros(20000, dtype=torch.bfloat16)
    for sizes, strides in [((2, 2, 16, 16), (1100, 528, 32)), ((3, 2, 16, 16), (512, 16, 32)), ((2, 2, 16, 16), (16, 32, 64)), ((1, 2, 16, 16), (7, 520, 32))]:
        strides = tuple(s // 8 * 8 for s in strides) + (1,)
        at = {sum(i * s for i, s in zip(ix, strides)) for ix in itertools.product(*map(range, sizes))}
        for shift in range(-2400, 2401, 8):
            a, b = buf.as_strided(sizes, strides, 4800), buf.as_strided(sizes, strides, 4800 + shift)
            shared = any(x + shift in at for x in at)
            with pytest.raises(RuntimeError) as e:
                K.kv_write(k, k, slots, a, b)
            told = "overlap" in str(e.value) or "one buffer" in str(e.value)
            assert told == shared, (sizes, strides, shift, str(e.value)[:100])
