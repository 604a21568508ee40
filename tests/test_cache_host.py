"""Refusals and the binding of the paged key/value cache: no GPU needed. The
caches here have no device (awa_cache_create_host); their memory is never read."""

from __future__ import annotations

import ctypes
import os
import re

import pytest
import torch

import awa_b200
from awa_b200 import cache as binding

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = binding._cache_library()
INVALID = -1
P = 4096  # an address that is aligned and never read


def params(**kw):
    p = dict(storage=awa_b200.AWA_BF16, heads=4, head_dim=128, page_tokens=16, pages=10, k=P, v=P,
             page_stride=4 * 16 * 128, head_stride=16 * 128, k_params=None, v_params=None, params_page_stride=0,
             params_head_stride=0)
    p.update(kw)
    return binding._CacheParams(**p)


def int4(**kw):
    return params(**{**dict(storage=awa_b200.AWA_INT4, page_stride=4 * 16 * 64, head_stride=16 * 64, k_params=P,
                            v_params=P, params_page_stride=4 * 16 * 4, params_head_stride=16 * 4), **kw})


def create(p):
    handle = ctypes.c_void_p()
    rc = LIB.awa_cache_create_host(ctypes.byref(p), ctypes.byref(handle))
    return rc, handle


@pytest.fixture
def cache():
    rc, handle = create(params())
    assert rc == 0
    yield handle
    LIB.awa_cache_destroy(handle)


def batch(**kw):
    b = dict(sequences=2, rows=5, max_rows=3, row_starts=P, past=P, page_table=P, table_width=4, table_stride=4)
    b.update(kw)
    return binding._CacheBatch(**b)


def error():
    return awa_b200.library().awa_last_error().decode()


def test_header_and_binding_agree():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "awa_cache.h")).read(), flags=re.S)
    declared = set(re.findall(r"\b(awa_\w+)\s*\(", text))
    assert declared == set(binding.CACHE_SYMBOLS)
    assert all(hasattr(LIB, name) for name in declared)


@pytest.mark.parametrize("p,word", [
    (params(storage=3), "storage"), (params(heads=0), "heads"), (params(heads=70000), "heads"),
    (params(pages=0), "pages"), (params(head_dim=0), "head_dim"), (params(head_dim=100), "head_dim"),
    (params(head_dim=136), "head_dim"), (params(page_tokens=8), "page_tokens"), (params(page_tokens=48), "page_tokens"),
    (params(page_tokens=512), "page_tokens"), (params(k=None), "NULL"), (params(head_stride=16 * 128 - 8), "strides"),
    (params(page_stride=3 * 16 * 128), "strides"), (params(k=P + 8), "16 bytes"),
    (params(page_stride=4 * 16 * 128 + 4), "16 bytes"), (int4(head_dim=96), "head_dim"), (int4(v_params=None), "NULL"),
    (int4(params_head_stride=16 * 4 - 8), "params"), (int4(k_params=P + 4), "params"),
    (params(page_stride=-4 * 16 * 128), "strides"),
])
def test_create_refuses(p, word):
    rc, handle = create(p)
    assert rc == INVALID and not handle.value and word in error()


def test_create_takes_either_order_of_pages_and_heads():
    for p in (params(), int4(), params(storage=awa_b200.AWA_F32), params(page_stride=16 * 128, head_stride=10 * 16 * 128)):
        rc, handle = create(p)
        assert rc == 0, error()
        LIB.awa_cache_destroy(handle)
    assert LIB.awa_cache_create_host(None, None) == INVALID
    LIB.awa_cache_destroy(None)


@pytest.mark.parametrize("b,word", [
    (batch(sequences=-1), "negative"), (batch(rows=-1), "negative"), (batch(max_rows=-2), "negative"),
    (batch(row_starts=None), "NULL"), (batch(past=None), "NULL"), (batch(page_table=None), "NULL"),
    (batch(table_stride=3), "table_stride"), (batch(table_width=1 << 28, table_stride=1 << 28), "2^30"), (batch(rows=1 << 30), "2^30"),
])
def test_batches_refused_by_every_call(cache, b, word):
    ref = ctypes.byref(b)
    for rc in (LIB.awa_cache_append(cache, ref, 0, 1, None, 0, P, 512, P, 512, None, 1, None, 0, None),
               LIB.awa_cache_read(cache, ref, 1, P, 512, P, 512, None),
               LIB.awa_cache_attention(cache, ref, 4, 1, P, 512, 1.0, 0, 0, 1, P, 512, None, 0, None)):
        assert rc == INVALID and word in error()
    assert LIB.awa_cache_attention_workspace_bytes(cache, ref, 4, 0, 0, 1) == 0


@pytest.mark.parametrize("kw,word", [
    (dict(in_dtype=2), "rows must be"), (dict(q_out_dtype=5), "rows must be"), (dict(k=None), "NULL"),
    (dict(q_out=None), "NULL"), (dict(q_heads=0), "q_heads"), (dict(qs=1023), "strides"), (dict(os_=100), "strides"),
    (dict(ks=511), "strides"), (dict(vs=511), "strides"), (dict(v=P + 1), "aligned"), (dict(q=P + 1), "aligned"),
    (dict(q_out=P, q=P, qs=2048), "q_out may be q"), (dict(rope=dict(table=None)), "rope"),
    (dict(rope=dict(table=P + 4)), "rope"), (dict(rope=dict(axes=0)), "rope"), (dict(rope=dict(axes=5)), "rope"),
    (dict(rope=dict(pairs=22)), "rope"), (dict(rope=dict(max_coord=0)), "rope"),
    (dict(), "without a device"), (dict(q=None, q_out=None, q_heads=0), "without a device"),
])
def test_append_refuses(cache, kw, word):
    a = dict(q_heads=8, in_dtype=1, q=2 * P, qs=1024, k=P, ks=512, v=P, vs=512, rope=None, q_out_dtype=1, q_out=P,
             os_=1024)
    a.update(kw)
    rope = None
    if a["rope"] is not None:
        rope = binding._CacheRope(**{**dict(table=P, max_coord=9, axes=3, pairs=21, coords=P), **a["rope"]})
    rc = LIB.awa_cache_append(cache, ctypes.byref(batch()), a["q_heads"], a["in_dtype"], a["q"], a["qs"], a["k"],
                              a["ks"], a["v"], a["vs"], None if rope is None else ctypes.addressof(rope),
                              a["q_out_dtype"], a["q_out"], a["os_"], None)
    assert rc == INVALID and word in error()


@pytest.mark.parametrize("kw,word", [
    (dict(out_dtype=2), "rows must be"), (dict(k=None), "NULL"), (dict(v=P + 1), "misaligned"), (dict(ks=511), "strides"),
    (dict(), "without a device"),
])
def test_read_refuses(cache, kw, word):
    a = {**dict(out_dtype=1, k=P, ks=512, v=P, vs=512), **kw}
    rc = LIB.awa_cache_read(cache, ctypes.byref(batch()), a["out_dtype"], a["k"], a["ks"], a["v"], a["vs"], None)
    assert rc == INVALID and word in error()


@pytest.mark.parametrize("kw,word", [
    (dict(heads=6), "q_heads"), (dict(heads=0), "q_heads"), (dict(dtype=0), "AWA_BF16"), (dict(q=None), "NULL"),
    (dict(out=None), "NULL"), (dict(q=P + 2), "16-byte"), (dict(qs=516), "16-byte"), (dict(qs=504), "strides"),
    (dict(os_=504), "strides"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(sinks=-1), "sinks"),
    (dict(window=-1), "window"), (dict(frame=0), "frame_tokens"), (dict(rows=1 << 29), "2^31"),
    (dict(), "without a device"), (dict(rows=0), "without a device"),
])
def test_attention_refuses(cache, kw, word):
    a = {**dict(heads=4, dtype=1, q=P, qs=512, scale=0.1, sinks=0, window=0, frame=1, out=P, os_=512, rows=5), **kw}
    rc = LIB.awa_cache_attention(cache, ctypes.byref(batch(rows=a["rows"])), a["heads"], a["dtype"], a["q"], a["qs"],
                                 a["scale"], a["sinks"], a["window"], a["frame"], a["out"], a["os_"], None, 0, None)
    assert rc == INVALID and word in error()


def test_null_handles():
    assert LIB.awa_cache_read(None, ctypes.byref(batch()), 1, P, 512, P, 512, None) == INVALID
    assert LIB.awa_cache_attention(None, None, 4, 1, P, 512, 1.0, 0, 0, 1, P, 512, None, 0, None) == INVALID
    assert LIB.awa_cache_attention_workspace_bytes(None, None, 4, 0, 0, 1) == 0


def host_cache(storage="bf16"):
    shape = (6, 2, 16)
    if storage == "int4":
        return awa_b200.KvCache(*(torch.zeros(shape + (64,), dtype=torch.uint8) for _ in range(2)),
                                *(torch.zeros(shape + (2, 2), dtype=torch.bfloat16) for _ in range(2)), host_only=True)
    return awa_b200.KvCache(*(torch.zeros(shape + (128,), dtype=torch.bfloat16) for _ in range(2)), host_only=True)


def test_python_refusals():
    ints = dict(dtype=torch.int32)
    starts, past, table = torch.zeros(3, **ints), torch.zeros(2, **ints), torch.zeros(2, 4, **ints)
    with pytest.raises(TypeError):
        awa_b200.CacheBatch(starts.long(), past, table, 0, 0)
    with pytest.raises(ValueError):
        awa_b200.CacheBatch(starts[:2], past, table, 0, 0)
    with pytest.raises(ValueError):
        awa_b200.CacheBatch(starts, past, table.T.contiguous().T, 0, 0)
    with pytest.raises(ValueError):
        awa_b200.CacheRope(torch.zeros(4, 3, 2).transpose(0, 1))
    with pytest.raises(ValueError):
        awa_b200.CacheRope(torch.zeros(4, 3, 2), torch.zeros(5, 3))
    k = torch.zeros(6, 2, 16, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        awa_b200.KvCache(k, k[:5], host_only=True)
    with pytest.raises(ValueError):
        awa_b200.KvCache(k, k, k, k, host_only=True)
    with pytest.raises(ValueError):
        awa_b200.KvCache(k.to(torch.uint8), k.to(torch.uint8), host_only=True)
    with pytest.raises(TypeError):
        awa_b200.KvCache(k.half(), k.half(), host_only=True)
    with pytest.raises(awa_b200.AwaError):
        awa_b200.KvCache(k[:, :, :12], k[:, :, :12], host_only=True)
    for cache in (host_cache(), host_cache("int4")):
        assert cache.head_dim == 128 and cache.heads == 2


def test_rope_table_is_exact_far_out():
    table = awa_b200.rope_table(3, 4, base=100.0, device="cpu")
    for c in range(3):
        for i in range(4):
            angle = torch.tensor(c * 100.0 ** (-i / 4), dtype=torch.float64)
            assert abs(table[c, i, 0].item() - angle.cos().item()) <= 2.0 ** -24
            assert abs(table[c, i, 1].item() - angle.sin().item()) <= 2.0 ** -24
