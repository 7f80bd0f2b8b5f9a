"""Generation on the fused engine: 16-bit weights, a paged key/value cache (16 or 8 bits), one CUDA graph per token.

``Decoder`` keeps the state of a batch of sequences: the cache's pages, the table that says which are whose, and the
lengths. ``append`` runs tokens through the model (prompts, or what a user adds later) and ``generate`` samples from it:

* prompts run through the fused blocks' kernels (attention over whole sequences) and leave K and V in the cache
  (``kv_write``); tokens added to sequences that have some read the cached ones back (``kv_read``) in front of them;
* a generated token is one row per sequence: ``kv_write``, then ``decode_attention`` over the sequence's pages;
* ``sample_tokens`` picks the next token on the device, from uniform numbers drawn beforehand, so that a step
  (about 10 launches a block) replays as one CUDA graph and nothing waits for the host.

Sequences may have unlike lengths. Pages are dealt out as sequences grow, from one pool for all.
"""
from __future__ import annotations

import contextlib
import functools
from typing import List, Optional, Sequence, Tuple

import torch

from ..ops import gemm as G
from ..ops import kernels as K
from ..ops._C import check_status
from .fused import LN_EPS, _dt, _is_moe, _vpad, fused_supported

GRAPH_STEPS = 8  # a capture costs some 5 steps: fewer are run one by one
MAX_VOCAB = 1 << 19  # of sample_tokens


def decoder_supported(model) -> Tuple[bool, str]:
    """Whether a ``Decoder`` takes this model, and why not (generate() on the plain modules takes any)."""
    topo = getattr(model, "topo", None)
    ok, why = fused_supported(model.cfg, topo)
    if not ok:
        return False, why
    if topo is not None and (getattr(topo, "tp", 1) > 1 or getattr(topo, "ep", 1) > 1):
        return False, "needs tp 1 and ep 1 (generate() on the plain modules has both)"
    if not hasattr(model.tr.ln_f.weight, "w16"):
        return False, "needs flattened parameters (parallel.flat.FlatParams)"
    if model.cfg.vocab_size > MAX_VOCAB:
        return False, f"samples from a vocabulary of at most {MAX_VOCAB}"
    return True, ""


def _on_its_device(method):
    """The method of a decoder with the decoder's device as the current one."""
    @functools.wraps(method)
    def call(self, *a, **kw):
        with torch.cuda.device(self.device) if self.device.type == "cuda" else contextlib.nullcontext():
            return method(self, *a, **kw)
    return call


def _capture(device: torch.device, fn):
    """The launches of ``fn`` on ``device``, the current one, as a graph; nothing runs yet.

    ``torch.cuda.graph`` would capture on one stream for the whole process, of the device that was current at the first capture:
    kernels for another device run at once then, and its graph is empty."""
    stream, g = torch.cuda.Stream(device), torch.cuda.CUDAGraph()
    torch.cuda.synchronize(device)
    torch.cuda.empty_cache()
    with torch.cuda.stream(stream):
        g.capture_begin()
        try:
            fn()
        finally:
            g.capture_end()
    return g


class Decoder:
    """State of ``batch`` sequences of a GPT on the fused engine.

    ``model``: a GPT whose parameters are flattened (``parallel.flat.FlatParams``), without tensor or expert
    parallelism. ``cache_bits`` 8 keeps K and V as signed codes with a power-of-two scale for each head of each token: half
    the memory and traffic, each value off by up to 1/127 of its head's largest. ``pages`` limits the pool (default: enough for
    ``block_size`` tokens of every sequence)."""

    def __init__(self, model, batch: int, cache_bits: int = 16, page_size: int = 64, pages: Optional[int] = None):
        cfg = model.cfg
        ok, why = decoder_supported(model)
        if not ok:
            raise ValueError(f"decoding on the fused engine: {why}")
        if cache_bits not in (8, 16):
            raise ValueError(f"a cache has 16 or 8 bits, got {cache_bits}")
        if batch < 1:
            raise ValueError("a decoder needs at least one sequence")
        self.model, self.batch, self.size = model, batch, page_size
        self.device, self.dtype = model.tr.wte.weight.device, _dt(model.tr.h[0])
        attn = model.tr.h[0].attn
        self.heads, self.dim = attn.nh_tp, attn.dh
        self.width = (cfg.block_size + page_size - 1) // page_size
        n_pages = batch * self.width if pages is None else pages
        shape = (cfg.n_layer, 2, n_pages, self.heads, page_size)
        kind = torch.int8 if cache_bits == 8 else self.dtype
        kv = torch.zeros(*shape, self.dim, device=self.device, dtype=kind)
        exps = torch.zeros(*shape, device=self.device, dtype=torch.uint8) if cache_bits == 8 else None
        self.pools = [dict(k_pages=kv[i, 0], v_pages=kv[i, 1], k_exp=None if exps is None else exps[i, 0],
                           v_exp=None if exps is None else exps[i, 1]) for i in range(cfg.n_layer)]
        self.free = list(range(n_pages - 1, -1, -1))
        self.owned: List[List[int]] = [[] for _ in range(batch)]
        self.lens = [0] * batch  # cached tokens of each sequence; the device has the same in self.lengths
        self.table = torch.zeros(batch, self.width, device=self.device, dtype=torch.int32)
        self.lengths = torch.zeros(batch, device=self.device, dtype=torch.int32)
        self.pending: Optional[torch.Tensor] = None  # the last sampled tokens [batch], not yet in the cache
        self.logits: Optional[torch.Tensor] = None   # of the next token [batch, padded vocabulary]

    # ---- pages ---------------------------------------------------------------
    def _reserve(self, more: Sequence[int]) -> None:
        """Pages for ``more[b]`` further tokens of sequence b, or an error that leaves everything as it was."""
        block = self.model.cfg.block_size
        want = [n + m for n, m in zip(self.lens, more)]
        if max(want) > block:
            raise ValueError(f"sequence of {max(want)} tokens > block_size {block}")
        need = [(w + self.size - 1) // self.size - len(o) for w, o in zip(want, self.owned)]
        if sum(n for n in need if n > 0) > len(self.free):
            raise ValueError(f"the cache has {len(self.free)} free pages of {self.size} tokens, "
                             f"{sum(n for n in need if n > 0)} are needed")
        if max(need) <= 0:
            return
        for b, n in enumerate(need):
            self.owned[b] += [self.free.pop() for _ in range(max(0, n))]
        rows = [o + [0] * (self.width - len(o)) for o in self.owned]
        self.table.copy_(torch.tensor(rows, dtype=torch.int32))

    def _slots(self, pos: torch.Tensor) -> torch.Tensor:
        """Slots of positions ``pos`` [batch, n] of the sequences."""
        page = self.table.gather(1, pos // self.size).long()
        return page * self.size + pos % self.size

    # ---- the model -----------------------------------------------------------
    def _mlp(self, blk, x: torch.Tensor) -> torch.Tensor:
        if _is_moe(blk):
            from .fused_moe import moe_sublayer_fwd
            return moe_sublayer_fwd(blk, None, x, False)[0]
        xn, _, _ = K.layernorm_fwd(x, blk.ln_2.weight, blk.ln_2.bias, LN_EPS, dtype=self.dtype)
        h, _ = G.linear_fwd_gelu(xn, blk.mlp.c_fc.weight.w16, blk.mlp.c_fc.bias)
        return G.linear_fwd_resid(h, blk.mlp.c_proj.weight.w16, blk.mlp.c_proj.bias, x)

    def _head(self, x: torch.Tensor) -> torch.Tensor:
        """fp32 [batch, H] -> logits [batch, padded vocabulary] in 16 bits."""
        tr, w = self.model.tr, self.model.lm_head.weight.w16
        xn, _, _ = K.layernorm_fwd(x, tr.ln_f.weight, tr.ln_f.bias, LN_EPS, dtype=self.dtype)
        return G.linear_fwd(xn, w, n=_vpad(self.model.cfg.vocab_size))

    def _blocks(self, x: torch.Tensor, slots: torch.Tensor, attend) -> torch.Tensor:
        """Every block on the rows of x (fp32), whose K and V go to ``slots``; attend(qkv, its layer) -> y."""
        for i, blk in enumerate(self.model.tr.h):
            attn = blk.attn
            xn, _, _ = K.layernorm_fwd(x, blk.ln_1.weight, blk.ln_1.bias, LN_EPS, dtype=self.dtype)
            qkv = G.linear_fwd(xn, attn.c_attn.weight.w16, attn.c_attn.bias)
            _, k, v = qkv.view(-1, 3, self.heads, self.dim).unbind(1)
            K.kv_write(k, v, slots, **self.pools[i])
            x = G.linear_fwd_resid(attend(qkv, i), attn.c_proj.weight.w16, attn.c_proj.bias, x)
            x = self._mlp(blk, x)
        return x

    def _step(self, tokens: torch.Tensor) -> torch.Tensor:
        """One token [batch] of every sequence -> logits of the next; device state only (captured)."""
        pos = self.lengths.long()
        tr = self.model.tr
        x = K.embedding_fwd(tokens.contiguous().view(1, -1), tr.wte.weight, tr.wpe.weight.index_select(0, pos))
        slots = self._slots(pos[:, None])[:, 0].contiguous()
        self.lengths += 1

        def attend(qkv, i):
            q = qkv.view(-1, 3, self.heads, self.dim)[:, 0]
            out, _ = K.decode_attention(q, table=self.table, lengths=self.lengths, **self.pools[i])
            return out.view(self.batch, -1)

        return self._head(self._blocks(x, slots, attend))

    # ---- what a user calls ---------------------------------------------------
    @torch.no_grad()
    @_on_its_device
    def append(self, idx: torch.Tensor, lengths: Optional[Sequence[int]] = None) -> torch.Tensor:
        """Adds ``idx`` [batch, n] to the sequences (``lengths[b]`` >= 1 of its first tokens, default all n; the others may be
        anything), behind what was generated last. Returns the logits [batch, vocabulary] of the token that follows each, in 16 bits."""
        if idx.dim() != 2 or idx.size(0) != self.batch or idx.size(1) < 1:
            raise ValueError(f"expected tokens [{self.batch}, n], got {tuple(idx.shape)}")
        lengths = [idx.size(1)] * self.batch if lengths is None else [int(n) for n in lengths]
        if len(lengths) != self.batch or min(lengths) < 1 or max(lengths) > idx.size(1):
            raise ValueError(f"lengths must be {self.batch} numbers from 1 to {idx.size(1)}")
        idx = idx[:, : max(lengths)].to(self.device)
        if self.pending is not None:
            idx, lengths = torch.cat([self.pending[:, None], idx], 1), [n + 1 for n in lengths]
        self._reserve(lengths)
        training = self.model.training
        self.model.eval()
        try:
            self.logits = self._prefill(idx.contiguous(), lengths)
        finally:
            self.model.train(training)
        self.pending = None
        self.lens = [a + n for a, n in zip(self.lens, lengths)]
        self.lengths.copy_(torch.tensor(self.lens, dtype=torch.int32))
        return self.logits[:, : self.model.cfg.vocab_size]

    def _prefill(self, idx: torch.Tensor, lengths: List[int]) -> torch.Tensor:
        B, S = idx.shape
        tr, dev = self.model.tr, self.device
        n = torch.tensor(lengths, device=dev)[:, None]
        at = torch.arange(S, device=dev)[None]
        old = self.lengths.long()[:, None]
        pos = (old + at).clamp_max_(self.model.cfg.block_size - 1)
        idx = torch.where(at < n, idx, 0)  # padding may be no token, whose row would be NaN: a weight of 0 does not take that out
        x = K.embedding_fwd(idx.view(1, -1), tr.wte.weight, tr.wpe.weight.index_select(0, pos.view(-1)))
        # tokens behind a sequence's own are rows like others, but leave nothing in the cache
        slots = torch.where(at < n, self._slots(pos), -1).view(-1)
        if max(self.lens) == 0:
            y = self._blocks(x, slots, lambda qkv, i: K.attention_fwd(qkv, B, S, self.heads, head_dim=self.dim)[0])
        else:
            # K and V of whole sequences come from the cache; q is put behind the cached tokens', of which nothing is asked
            T = max(a + m for a, m in zip(self.lens, lengths))
            every = torch.arange(T, device=dev)[None].expand(B, T)
            held = torch.where(every < old + n, self._slots(every), -1).reshape(-1)
            rows = (torch.arange(B, device=dev)[:, None] * T + (old + at).clamp_max_(T - 1)).view(-1)
            keep = (at < n).view(-1, 1, 1)

            def attend(qkv, i):
                full = torch.zeros(B * T, 3, self.heads, self.dim, device=dev, dtype=qkv.dtype)
                full[:, 1], full[:, 2] = K.kv_read(held, **self.pools[i], dtype=qkv.dtype)
                q = qkv.view(-1, 3, self.heads, self.dim)[:, 0]
                full[:, 0].index_add_(0, rows, torch.where(keep, q, torch.zeros_like(q)))  # (clamped rows add 0)
                y, _ = K.attention_fwd(full.view(B * T, -1), B, T, self.heads, head_dim=self.dim)
                return y.index_select(0, rows)

            y = self._blocks(x, slots, attend)
        return self._head(y.view(B, S, -1)[torch.arange(B, device=dev), n[:, 0] - 1].contiguous())

    def _check(self, tokens: torch.Tensor) -> None:
        """An error where a sequence got no token (``tokens`` [steps, batch]); waits for the device."""
        broken = (tokens < 0).any(0).nonzero()[:, 0].tolist()
        if not broken:
            return
        text = f"no token for sequences {broken}: their logits hold NaN or +inf, or nothing but -inf"
        if self.device.type == "cuda":  # what the steps behind such a token made of it is reported here, and not later
            try:
                check_status(self.device.index)
            except RuntimeError as e:
                raise RuntimeError(text) from e
        raise RuntimeError(text)

    @torch.no_grad()
    @_on_its_device
    def generate(self, n: int, temperature: float = 1.0, top_k: Optional[int] = None, top_p: float = 1.0, min_p: float = 0.0,
                 generator: Optional[torch.Generator] = None, cuda_graph: bool = True) -> torch.Tensor:
        """``n`` sampled tokens of every sequence, [batch, n] (``temperature`` <= 0: the most likely ones).

        The settings are ``sample_tokens``'s. The last one is run through the model when more is generated or appended. Logits
        that give no token (NaN, say) are an error; it leaves the sequences as they were."""
        if self.logits is None and self.pending is None:
            raise ValueError("append a prompt first")
        if n < 1:
            return torch.empty(self.batch, 0, dtype=torch.long, device=self.device)
        steps = n if self.logits is None else n - 1
        if max(self.lens) + steps + 1 > self.model.cfg.block_size:
            raise ValueError(f"sequence of {max(self.lens) + steps + 1} tokens > block_size {self.model.cfg.block_size}")
        self._reserve([steps] * self.batch)
        V = self.model.cfg.vocab_size
        u = torch.rand(n, self.batch, device=self.device, generator=generator)
        out = torch.empty(n, self.batch, dtype=torch.long, device=self.device)
        at = torch.zeros(1, dtype=torch.long, device=self.device)
        settings = dict(temperature=float(temperature), top_k=int(top_k or 0), top_p=float(top_p), min_p=float(min_p))

        def sample(logits):
            token = K.sample_tokens(logits, V, u.index_select(0, at)[0], **settings)
            out.index_copy_(0, at, token[None])
            at.add_(1)
            return token

        training, logits = self.model.training, self.logits
        self.model.eval()
        try:
            if logits is not None:
                token = sample(logits)
                self.logits = None
            else:
                token = self.pending
            graph = cuda_graph and self.device.type == "cuda" and steps >= GRAPH_STEPS
            eager = 1 if graph else steps  # with a graph: one step to warm up
            for _ in range(eager):
                token = sample(self._step(token))
            if graph:
                token = token.clone()
                g = _capture(self.device, lambda: token.copy_(sample(self._step(token))))
                for _ in range(steps - eager):
                    g.replay()
                torch.cuda.current_stream().synchronize()  # before the graph and its memory go
                del g
            self._check(out)
        except BaseException:  # nothing was generated: the next call begins where this one did
            self.logits = logits
            self.lengths.copy_(torch.tensor(self.lens, dtype=torch.int32))
            raise
        finally:
            self.model.train(training)
        self.lens = [a + steps for a in self.lens]
        self.pending = token.clone()
        return out.t().contiguous()
