"""Arguments of the paged key/value cache that have to be refused before any
kernel sees them, and what a call asks for: no GPU needed."""

from __future__ import annotations

import ctypes
import glob
import os
import re

import pytest
import torch

import awa_b200
from awa_b200 import cache as binding

INTS = dict(dtype=torch.int32)


@pytest.mark.parametrize("table", [
    torch.zeros(4, **INTS).expand(3, -1),                       # one row for all: stride 0
    torch.zeros(6, **INTS).as_strided((3, 4), (1, 1)),          # rows that overlap
    torch.zeros(9, **INTS).as_strided((3, 4), (2, 1)),
], ids=["expanded", "stride1", "stride2"])
def test_page_tables_whose_rows_overlap(table):
    """Passed on with a stride of the width, such a table would be read behind its storage."""
    with pytest.raises(ValueError, match="page_table"):
        awa_b200.CacheBatch(torch.zeros(4, **INTS), torch.zeros(3, **INTS), table, 3, 1)


def test_strides_of_page_tables_that_are_taken():
    starts, past = torch.zeros(4, **INTS), torch.zeros(3, **INTS)
    wide = torch.zeros(3, 9, **INTS)
    assert awa_b200.CacheBatch(starts, past, wide[:, 2:6], 3, 1).c.table_stride == 9
    assert awa_b200.CacheBatch(starts, past, wide, 3, 1).c.table_stride == 9
    # the stride of a single row is never used
    one = torch.zeros(4, **INTS).expand(1, -1).as_strided((1, 4), (0, 1))
    assert awa_b200.CacheBatch(starts[:2], past[:1], one, 3, 1).c.table_stride == 4


def test_pages_in_host_memory_are_refused():
    k = torch.zeros(6, 2, 16, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        awa_b200.KvCache(k, k.clone())


class OnDevice:
    """A tensor's stand-in that lies on a GPU that need not be there."""

    def __init__(self, index):
        self.device, self.dtype, self.shape = torch.device("cuda", index), torch.bfloat16, (6, 2, 16, 128)

    def dim(self):
        return 4

    def stride(self, i=None):
        strides = (2 * 16 * 128, 16 * 128, 128, 1)
        return strides if i is None else strides[i]

    def data_ptr(self):
        return 4096


def test_a_handle_is_made_on_the_device_of_its_pages(monkeypatch):
    """awa_cache_create takes the current device: the pages' one has to be that."""
    current, made_on = [0], []

    class Device:
        def __init__(self, device):
            self.index = torch.device(device).index

        def __enter__(self):
            current.append(self.index)

        def __exit__(self, *_):
            current.pop()

    class Library:
        def awa_cache_create(self, params, handle):
            made_on.append(current[-1])
            return 0

        def awa_cache_destroy(self, handle):
            pass

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(binding, "_lib", Library())
    cache = awa_b200.KvCache(OnDevice(1), OnDevice(1))
    assert made_on == [1] and current == [0]
    assert cache.device.index == 1
    with pytest.raises(ValueError, match="one device"):
        awa_b200.KvCache(OnDevice(1), OnDevice(0))


def host_cache(storage="bf16", pages=6, heads=2, page=16, dim=128):
    shape = (pages, heads, page)
    with torch.device("meta"):  # never read: pages of any number cost nothing
        if storage == "int4":
            tensors = [torch.empty(shape + (dim // 2,), dtype=torch.uint8) for _ in range(2)]
            tensors += [torch.empty(shape + (dim // 64, 2), dtype=torch.bfloat16) for _ in range(2)]
        else:
            tensors = [torch.empty(shape + (dim,), dtype=torch.bfloat16) for _ in range(2)]
    return awa_b200.KvCache(*(Meta(t) for t in tensors), host_only=True)


class Meta:
    """A meta tensor with an address."""

    def __init__(self, t):
        self._t = t
        self.device, self.dtype, self.shape, self.stride, self.dim = t.device, t.dtype, t.shape, t.stride, t.dim

    def data_ptr(self):
        return 4096


def host_batch(sequences, width, rows, max_rows):
    return awa_b200.CacheBatch(torch.empty(sequences + 1, **INTS), torch.empty(sequences, **INTS),
                               torch.empty(sequences, width, **INTS), rows, max_rows)


@pytest.mark.parametrize("make", [
    lambda n: torch.zeros(1, dtype=torch.uint8).expand(n),
    lambda n: torch.zeros(4 * n, dtype=torch.uint8)[::4],
    lambda n: torch.zeros(n // 256, 1, dtype=torch.uint8).expand(-1, 257),
], ids=["expanded", "strided", "rows"])
def test_workspaces_with_less_memory_than_elements(make):
    k = torch.zeros(6, 2, 16, 128, dtype=torch.bfloat16)
    cache, batch = awa_b200.KvCache(k, k, host_only=True), host_batch(1, 6, 90, 90)
    need = cache.attention_workspace_bytes(batch, 4)
    assert need > 0
    q = torch.zeros(90, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="contiguous"):
        cache.attention(batch, q, workspace=make(need + 256))


def test_no_wait_reports_the_code_of_a_bad_batch():
    """A wait that ran out must not look like a bad page or coordinate."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    codes = set()
    for path in glob.glob(os.path.join(root, "seedvr2-ncnn_b200", "csrc", "*.cu")):
        for line in open(path):
            codes.update(int(c) for c in re.findall(r"(?:error_flag|wait\(.*),\s*(\d\d)\)", line))
    assert {73, 79, 80, 92, 31, 61} <= codes  # the sources were understood
    assert not codes & {awa_b200.AWA_CACHE_BAD_PAGE, awa_b200.AWA_CACHE_BAD_COORD}


@pytest.mark.parametrize("window,frame", [(2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31 - 1, 1), (1, 2 ** 31 - 1), (2 ** 20, 2 ** 30)])
@pytest.mark.parametrize("sinks", [0, 2 ** 31 - 1])
@pytest.mark.parametrize("sequences", [1, 33, 64, 5000])
@pytest.mark.parametrize("storage", ["bf16", "int4"])
def test_a_window_without_end_needs_no_more_than_none(window, frame, sinks, sequences, storage):
    """Any product of window and frame is taken: past the table's reach it is all the same."""
    cache, batch = host_cache(storage), host_batch(sequences, 40, 90 * sequences, 90)
    most = cache.attention_workspace_bytes(batch, 4)
    assert 0 < cache.attention_workspace_bytes(batch, 4, sinks, window, frame) <= most


def test_rows_at_a_frame_s_edge_count_both_frames():
    """A window of one frame of 1200: two rows either side of an edge see 2400 keys, more
    than a cluster of blocks is for (2048), so the parts of several blocks need a workspace."""
    cache, batch = host_cache(), host_batch(1, 1000, 2, 2)
    assert cache.attention_workspace_bytes(batch, 2, 0, 1, 1200) > 0
    assert cache.attention_workspace_bytes(batch, 2, 0, 1, 900) == 0  # 1800 keys


@pytest.mark.parametrize("field", ["row_starts", "past", "page_table", "coords"])
@pytest.mark.parametrize("off", [1, 2])
def test_index_arrays_off_their_alignment(field, off):
    """A kernel's load from such an address would fault."""
    lib, P = awa_b200.library(), 4096
    cache = host_cache()
    arrays = dict(row_starts=P, past=P, page_table=P, coords=P)
    arrays[field] += off
    batch = binding._CacheBatch(2, 5, 3, arrays["row_starts"], arrays["past"], arrays["page_table"], 4, 4)
    rope = binding._CacheRope(P, 9, 3, 21, arrays["coords"])
    calls = [lib.awa_cache_append(cache._handle, ctypes.byref(batch), 0, 1, None, 0, P, 256, P, 256,
                                  ctypes.byref(rope), 1, None, 0, None)]
    if field != "coords":
        calls += [lib.awa_cache_read(cache._handle, ctypes.byref(batch), 1, P, 256, P, 256, None),
                  lib.awa_cache_attention(cache._handle, ctypes.byref(batch), 4, 1, P, 512, 1.0, 0, 0, 1, P, 512, None, 0,
                                          None)]
    assert calls == [awa_b200.AWA_ERR_INVALID] * len(calls)
    assert "aligned" in lib.awa_last_error().decode()


@pytest.mark.parametrize("name", ["sinks", "window", "frame_tokens"])
@pytest.mark.parametrize("value", [2 ** 31, 2 ** 32, 2 ** 32 + 1, 2 ** 63 - 1, -2 ** 32 + 1])
def test_masks_that_do_not_fit_an_int(name, value):
    """ctypes would cut them to 32 bits: a prefix of 2^32 + 4 rows to one of 4."""
    cache, batch = host_cache(), host_batch(1, 6, 2, 2)
    k = torch.zeros(6, 2, 16, 128, dtype=torch.bfloat16)
    small = awa_b200.KvCache(k, k, host_only=True)
    with pytest.raises(ValueError, match=name):
        small.attention(batch, torch.zeros(2, 4, 128, dtype=torch.bfloat16), **{name: value})
    with pytest.raises(ValueError, match=name):
        cache.attention_workspace_bytes(batch, 4, **{name: value})


def test_row_counts_that_do_not_fit_an_int():
    for rows, most in ((2 ** 32 + 2, 2), (2, 2 ** 32 + 2), (2, 2 ** 31)):
        with pytest.raises(ValueError, match="rows"):
            host_batch(1, 6, rows, most)


GIB = 2 ** 30


@pytest.mark.parametrize("pages,heads,page,sequences,width", [
    (2000, 8, 64, 64, 512),      # streams of a few hundred tokens with room for 32768 in the table
    (100, 2, 16, 1000, 4000),
    (40000, 8, 64, 64, 512),     # a cache that could be full of what they see
    (1000000, 20, 64, 3, 300000),
    (5000, 1, 256, 200, 4096),
])
def test_workspace_of_many_rows_over_4_bits(pages, heads, page, sequences, width):
    """Pools of fp16 pages: never more of them than the cache has, and those of as
    many heads at a time as 1 GiB holds (one, if one head's are more)."""
    cache = host_cache("int4", pages, heads, page)
    batch = host_batch(sequences, width, 9 * sequences, 9)
    one_head = min(pages, sequences * width) * page * 128 * 2 * 2
    beside = sequences * width * 4 + 9 * sequences * 4 * heads * (128 * 2 + 4) + (80 << 20)  # table, q, parts of rows
    assert cache.attention_workspace_bytes(batch, 4 * heads) <= max(min(2 * GIB, heads * one_head), one_head) + beside


@pytest.mark.parametrize("storage,field", [
    (s, f + "_stride") for s in ("bf16", "f32", "int4")
    for f in ("page", "head", *(("params_page", "params_head") if s == "int4" else ()))])
@pytest.mark.parametrize("value", [2 ** 40, 2 ** 60, 2 ** 62, 2 ** 63 - 2 ** 10])
def test_strides_that_no_memory_has(storage, field, value):
    """Their products would pass 64 bits, and tensor maps end at 2^40 bytes."""
    four = storage == "int4"
    row = 64 if four else 128
    p = dict(page_stride=4 * 16 * row, head_stride=16 * row, params_page_stride=4 * 16 * 4, params_head_stride=16 * 4)
    p[field] = value
    code = {"bf16": awa_b200.AWA_BF16, "f32": awa_b200.AWA_F32, "int4": awa_b200.AWA_INT4}[storage]
    params = binding._CacheParams(code, 4, 128, 16, 10, 4096, 4096, p["page_stride"], p["head_stride"],
                                  4096 if four else None, 4096 if four else None, p["params_page_stride"],
                                  p["params_head_stride"])
    handle = ctypes.c_void_p()
    rc = awa_b200.library().awa_cache_create_host(ctypes.byref(params), ctypes.byref(handle))
    awa_b200.library().awa_cache_destroy(handle)
    assert rc == awa_b200.AWA_ERR_INVALID
