"""Refusals of the decoding operators: every check of arguments precedes the look at the device, so they show without one."""
import math

import pytest
import torch

from heiretsu_b200.ops import _C
from heiretsu_b200.ops import kernels as K

pytestmark = pytest.mark.skipif(not _C.available(), reason="the extension is not built")

BF16, F16 = torch.bfloat16, torch.float16


def _pools(pages=4, heads=2, size=16, dim=64, dtype=BF16):
    p = {n: torch.zeros(pages, heads, size, dim, dtype=dtype) for n in ("k_pages", "v_pages")}
    if dtype == torch.int8:
        p |= {n: torch.zeros(pages, heads, size, dtype=torch.uint8) for n in ("k_exp", "v_exp")}
    return p


def _refused(match, fn, *a, **kw):
    with pytest.raises((RuntimeError, TypeError), match=match):
        fn(*a, **kw)


def _offset(t, n):
    """The same tensor, n elements behind a 16-byte boundary."""
    out = torch.zeros(t.numel() + n, dtype=t.dtype)[n:].view(t.shape)
    return out.copy_(t)


def test_caches_that_are_refused():
    slots = torch.arange(3)
    k = torch.zeros(3, 2, 64, dtype=BF16)
    for match, pools in [
        ("head dim must be", _pools(dim=48)), ("head dim must be", _pools(dim=256)), ("page size", _pools(size=8)),
        ("page size", _pools(size=24)), ("dtype of the tokens", _pools(dtype=F16)), ("bf16, fp16 or, in 8 bits", _pools(dtype=torch.float32)),
        ("no other, has", _pools() | {"k_exp": torch.zeros(4, 2, 16, dtype=torch.uint8)}),
        ("no other, has", {n: t for n, t in _pools(dtype=torch.int8).items() if n != "v_exp"}),
        ("uint8", _pools(dtype=torch.int8) | {"v_exp": torch.zeros(4, 2, 16, dtype=torch.int8)}),
        ("uint8", _pools(dtype=torch.int8) | {"v_exp": torch.zeros(4, 2, 17, dtype=torch.uint8)}),
        ("uint8", _pools(dtype=torch.int8) | {"v_exp": torch.zeros(4, 2, 1, dtype=torch.uint8).expand(4, 2, 16)}),
        ("must both be", _pools() | {"v_pages": torch.zeros(4, 2, 16, 32, dtype=BF16)}),
        ("one dtype", _pools() | {"v_pages": torch.zeros(4, 2, 16, 64, dtype=F16)}),
        ("no two slots overlap", _pools() | {"v_pages": torch.zeros(4, 1, 16, 64, dtype=BF16).expand(4, 2, 16, 64)}),
        ("contiguous", _pools() | {"v_pages": torch.zeros(4, 2, 64, 16, dtype=BF16).transpose(2, 3)}),
        ("16-byte", _pools() | {"v_pages": _offset(_pools()["v_pages"], 1)}),
        ("16-byte", _pools() | {"v_pages": torch.zeros(4, 2, 16, 68, dtype=BF16)[..., :64]}),
        ("must not be one buffer", dict.fromkeys(("k_pages", "v_pages"), _pools()["k_pages"])),
    ]:
        _refused(match, K.kv_write, k, k, slots, **pools)
        if "dtype of the tokens" not in match:
            _refused(match, K.kv_read, slots, **pools)
        _refused(match, K.decode_attention, k[:1], table=torch.zeros(1, 1, dtype=torch.int32), lengths=torch.zeros(1, dtype=torch.int32),
                 **pools)


def test_tokens_that_are_refused():
    k, slots, pools = torch.zeros(3, 2, 64, dtype=BF16), torch.arange(3), _pools()
    for match, a in [
        ("bf16 or fp16", (k.float(), k.float(), slots)), ("bf16 or fp16", (k, k.half(), slots)), ("int64", (k, k, slots.int())),
        ("int64", (k, k, torch.arange(6)[::2])), ("int64", (k, k, slots[None])), ("of the slots and the cache", (k, k, torch.arange(4))),
        ("of the slots and the cache", (k[:, :1], k[:, :1], slots)), ("of the slots and the cache", (k[..., :32], k[..., :32], slots)),
        ("of the slots and the cache", (k, k[:2], slots)),
        ("channels of k and v", (torch.zeros(3, 64, 2, dtype=BF16).transpose(1, 2), k, slots)),
        ("CUDA", (k, k, slots)),
    ]:
        _refused(match, K.kv_write, *a, **pools)
    _refused("its own dtype", K.kv_read, slots, **pools, dtype=F16)
    _refused("bf16, fp16 or fp32", K.kv_read, slots, **_pools(dtype=torch.int8), dtype=torch.float64)
    _refused("int64", K.kv_read, slots.int(), **pools)
    _refused("CUDA", K.kv_read, slots, **pools)
    _refused("CUDA", K.kv_read, slots, **_pools(dtype=torch.int8), dtype=torch.float32)


def test_queries_that_are_refused():
    pools, q = _pools(), torch.zeros(3, 4, 64, dtype=BF16)
    table, n = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for match, q_, t, ln, kw in [
        ("bf16 or fp16", q.float(), table, n, {}), ("dtype of the tokens", q.half(), table, n, {}),
        ("head dim of the cache", q[..., :32], table, n, {}), ("head dim of the cache", q[0], table, n, {}),
        ("head dim of the cache", torch.zeros(3, 64, 4, dtype=BF16).transpose(1, 2), table, n, {}),
        ("multiple of the cache's", q[:, :3], table, n, {}), ("multiple of the cache's", q[:, :0], table, n, {}),
        ("table", q, table.long(), n, {}), ("table", q, table[:2], n, {}), ("table", q, torch.zeros(2, 3, dtype=torch.int32).t(), n, {}),
        ("lengths", q, table, n.long(), {}), ("lengths", q, table, n[:2], {}), ("lengths", q, table, torch.zeros(6, dtype=torch.int32)[::2], {}),
        ("finite", q, table, n, {"scale": math.inf}), ("finite", q, table, n, {"scale": math.nan}), ("CUDA", q, table, n, {}),
    ]:
        _refused(match, K.decode_attention, q_, table=t, lengths=ln, **pools, **kw)


def test_logits_that_are_refused():
    x, u = torch.zeros(3, 100), torch.zeros(3)
    for match, x_, V, u_, kw in [
        ("bf16, fp16 or fp32", x.double(), 100, u, {}), ("2-D", x[0], 100, u, {}), ("2-D", torch.zeros(100, 3).t(), 100, u, {}),
        (r"V must be in", x, 101, u, {}), (r"V must be in", x, 0, u, {}), ("at most 524288", torch.zeros(1, 2 ** 19 + 1), 2 ** 19 + 1, u[:1], {}),
        ("u \\(fp32", x, 100, u.double(), {}), ("u \\(fp32", x, 100, u[:2], {}), ("u \\(fp32", x, 100, torch.zeros(6)[::2], {}),
        ("temperature", x, 100, u, {"temperature": u.double()}), ("top_k", x, 100, u, {"top_k": torch.zeros(3, dtype=torch.int32)}),
        ("top_p", x, 100, u, {"top_p": u[:1]}), ("min_p", x, 100, u, {"min_p": u[None]}), ("not a number", x, 100, u, {"top_p": math.nan}),
        ("not a number", x, 100, u, {"temperature": math.nan}), ("CUDA", x, 100, u, {}),
    ]:
        _refused(match, K.sample_tokens, x_, V, u_, **kw)
