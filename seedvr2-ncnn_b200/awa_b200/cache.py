"""Paged key/value cache (include/awa_cache.h): rows appended with the position
rotation applied on the way, attention over the cache with a sliding window and
a prefix that stays visible, storage in fp32, bf16 or 4 bits.

    cache = KvCache.empty(pages=1000, page_tokens=64, heads=20, head_dim=128)
    batch = CacheBatch(row_starts, past, page_table, rows, max_rows)   # device int32 tensors
    q = cache.append(batch, k, v, q=q, rope=CacheRope(rope_table(4096, 21), coords))
    out = cache.attention(batch, q, sinks=58, window=5, frame_tokens=4096)

The caller owns the memory and hands out the pages. Lengths and page numbers
live in device tensors, so a captured step serves later ones when they change.
"""

from __future__ import annotations

import ctypes
from typing import Optional

from . import AWA_BF16, AWA_F32, _check, _dtype_code, _torch, library

AWA_INT4 = 2
AWA_CACHE_GROUP = 64  # features that share a scale and a minimum in a 4-bit cache
AWA_CACHE_BAD_PAGE = 71
AWA_CACHE_BAD_COORD = 72

_INTS = 2 ** 31  # a C int holds -_INTS .. _INTS - 1

# Every symbol declared in include/awa_cache.h.
CACHE_SYMBOLS = (
    "awa_cache_create", "awa_cache_create_host", "awa_cache_destroy", "awa_cache_append", "awa_cache_read",
    "awa_cache_attention_workspace_bytes", "awa_cache_attention",
)


class _CacheParams(ctypes.Structure):
    _fields_ = [("storage", ctypes.c_int), ("heads", ctypes.c_int), ("head_dim", ctypes.c_int),
                ("page_tokens", ctypes.c_int), ("pages", ctypes.c_int), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("page_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64), ("k_params", ctypes.c_void_p),
                ("v_params", ctypes.c_void_p), ("params_page_stride", ctypes.c_int64),
                ("params_head_stride", ctypes.c_int64)]


class _CacheBatch(ctypes.Structure):
    _fields_ = [("sequences", ctypes.c_int), ("rows", ctypes.c_int), ("max_rows", ctypes.c_int),
                ("row_starts", ctypes.c_void_p), ("past", ctypes.c_void_p), ("page_table", ctypes.c_void_p),
                ("table_width", ctypes.c_int), ("table_stride", ctypes.c_int64)]


class _CacheRope(ctypes.Structure):
    _fields_ = [("table", ctypes.c_void_p), ("max_coord", ctypes.c_int), ("axes", ctypes.c_int),
                ("pairs", ctypes.c_int), ("coords", ctypes.c_void_p)]


_lib = None


def _cache_library():
    global _lib
    if _lib is None:
        lib = library()
        i, p, i64, sz = ctypes.c_int, ctypes.c_void_p, ctypes.c_int64, ctypes.c_size_t
        for name, (res, args) in {
            "awa_cache_create": (i, [p, ctypes.POINTER(p)]),
            "awa_cache_create_host": (i, [p, ctypes.POINTER(p)]),
            "awa_cache_destroy": (None, [p]),
            "awa_cache_append": (i, [p, p, i, i, p, i64, p, i64, p, i64, p, i, p, i64, p]),
            "awa_cache_read": (i, [p, p, i, p, i64, p, i64, p]),
            "awa_cache_attention_workspace_bytes": (sz, [p, p, i, i, i, i]),
            "awa_cache_attention": (i, [p, p, i, i, p, i64, ctypes.c_float, i, i, i, p, i64, p, sz, p]),
        }.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


def _current_raw_stream(index: int) -> int:
    """cudaStream_t of the current stream of a device."""
    torch = _torch()
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return torch.cuda.current_stream(index).cuda_stream if raw is None else raw(index)


def _check_mask(sinks, window, frame_tokens):
    """ctypes cuts an int to 32 bits; what is left could be a valid mask."""
    if not (-_INTS <= sinks < _INTS and -_INTS <= window < _INTS and -_INTS <= frame_tokens < _INTS):
        raise ValueError(f"sinks ({sinks}), window ({window}) and frame_tokens ({frame_tokens}) must fit 32 bits")


def rope_table(max_coord: int, pairs: int, base: float = 10000.0, device="cuda"):
    """[max_coord, pairs, 2] fp32 (cos, sin) of coord * base^(-i / pairs), the
    angles in float64 (exact where fp32 angles of far positions are not)."""
    torch = _torch()
    rates = torch.pow(float(base), -torch.arange(pairs, dtype=torch.float64, device=device) / pairs)
    angle = torch.arange(max_coord, dtype=torch.float64, device=device)[:, None] * rates
    return torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()


class CacheRope:
    """The rotation of q and k rows (awa_cache_rope): `table` [max_coord, pairs,
    2] fp32 (cos, sin), `coords` [rows, axes] int32 or None (one axis: the
    row's position in its sequence)."""

    def __init__(self, table, coords=None):
        torch = _torch()
        if table.dim() != 3 or table.shape[2] != 2 or table.dtype != torch.float32 or not table.is_contiguous():
            raise ValueError("a rope table is a contiguous fp32 [max_coord, pairs, 2] tensor")
        if coords is not None and (coords.dim() != 2 or coords.dtype != torch.int32 or not coords.is_contiguous() or
                                   coords.device != table.device):
            raise ValueError("coords is a contiguous int32 [rows, axes] tensor on the table's device")
        self.table, self.coords = table, coords
        self.rows = None if coords is None else coords.shape[0]
        self.c = _CacheRope(table.data_ptr(), table.shape[0], 1 if coords is None else coords.shape[1],
                            table.shape[1], None if coords is None else coords.data_ptr())
        self.ref = ctypes.addressof(self.c)


class CacheBatch:
    """One step's rows (awa_cache_batch): row_starts [sequences + 1], past
    [sequences], page_table [sequences, width], int32 on the device. `rows` is
    the number of rows of the row tensors, `max_rows` the most of one sequence
    (chooses the kernel). The tensors' contents may change between calls."""

    def __init__(self, row_starts, past, page_table, rows: int, max_rows: int):
        torch = _torch()
        if any(t.dtype != torch.int32 for t in (row_starts, past, page_table)):
            raise TypeError("row_starts, past and page_table are int32")
        if (past.dim() != 1 or row_starts.dim() != 1 or page_table.dim() != 2 or
                row_starts.shape[0] != past.shape[0] + 1 or page_table.shape[0] != past.shape[0]):
            raise ValueError("row_starts [sequences + 1], past [sequences] and page_table [sequences, width] expected")
        if (row_starts.stride(0) != 1 or (past.shape[0] > 1 and past.stride(0) != 1) or
                (page_table.shape[1] > 1 and page_table.stride(1) != 1)):
            raise ValueError("row_starts, past and the rows of page_table must be dense")
        if past.shape[0] > 1 and page_table.stride(0) < page_table.shape[1]:
            raise ValueError("the rows of page_table must not overlap (an expanded table: .contiguous())")
        if not row_starts.device == past.device == page_table.device:
            raise ValueError("row_starts, past and page_table must be on one device")
        self.row_starts, self.past, self.page_table = row_starts, past, page_table
        self.rows, self.device = int(rows), past.device
        if not (0 <= rows < _INTS and 0 <= max_rows < _INTS):
            raise ValueError(f"rows ({rows}) and max_rows ({max_rows}) must be 0 or more and fit 32 bits")
        # a single row's stride is never used, but has to hold a row
        width = page_table.shape[1]
        self.c = _CacheBatch(past.shape[0], self.rows, int(max_rows), row_starts.data_ptr(), past.data_ptr(),
                             page_table.data_ptr(), width, max(page_table.stride(0), width))
        self.ref = ctypes.addressof(self.c)


class KvCache:
    """A cache over the caller's pages: k, v [pages, heads, page_tokens,
    head_dim] bf16 or fp32, or uint8 [..., head_dim / 2] with k_params, v_params
    bf16 [pages, heads, page_tokens, head_dim / 64, 2] (scale, minimum) for 4
    bits. k and v may be views with other page and head strides (the same for
    both). The handle belongs to their device, which has to be current in the
    calls. host_only: a handle that only checks arguments (awa_cache_create_host)."""

    def __init__(self, k, v, k_params=None, v_params=None, host_only: bool = False):
        torch = _torch()
        lib = _cache_library()
        four = k.dtype == torch.uint8
        storage = AWA_INT4 if four else _dtype_code(k)
        tensors = [k, v] + ([k_params, v_params] if four else [])
        if four != (k_params is not None) or four != (v_params is not None):
            raise ValueError("k_params and v_params belong to a uint8 (4-bit) cache, and only to one")
        if k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype or v.stride() != k.stride():
            raise ValueError("k and v are [pages, heads, page_tokens, head_dim] with equal strides and dtype")
        if any(t.device != k.device for t in tensors):
            raise ValueError("the cache's tensors must be on one device")
        if not host_only and k.device.type != "cuda":
            raise ValueError("the cache's tensors must be CUDA tensors")
        pages, heads, page_tokens, row = k.shape
        self.head_dim = row * 2 if four else row
        if k.stride(3) != 1 or k.stride(2) != row:
            raise ValueError("the rows of a page must be dense")
        params = _CacheParams(storage, heads, self.head_dim, page_tokens, pages, k.data_ptr(), v.data_ptr(),
                              k.stride(0), k.stride(1), None, None, 0, 0)
        if four:
            groups = self.head_dim // AWA_CACHE_GROUP
            for t in (k_params, v_params):
                if (t.dtype != torch.bfloat16 or t.shape != (pages, heads, page_tokens, groups, 2) or
                        t.stride()[2:] != (2 * groups, 2, 1) or t.stride() != k_params.stride()):
                    raise ValueError("params are bf16 [pages, heads, page_tokens, head_dim / 64, 2], dense in a page")
            params.k_params, params.v_params = k_params.data_ptr(), v_params.data_ptr()
            params.params_page_stride, params.params_head_stride = k_params.stride(0), k_params.stride(1)
        handle = ctypes.c_void_p()
        if host_only:
            _check(lib.awa_cache_create_host(ctypes.byref(params), ctypes.byref(handle)))
        else:
            with torch.cuda.device(k.device):  # the handle belongs to the current device
                _check(lib.awa_cache_create(ctypes.byref(params), ctypes.byref(handle)))
        self._handle = handle.value
        self.k, self.v, self.k_params, self.v_params = k, v, k_params, v_params
        self.heads, self.storage, self.device = heads, storage, k.device
        self._type = AWA_F32 if storage == AWA_F32 else AWA_BF16
        self._rows_dtype = torch.float32 if storage == AWA_F32 else torch.bfloat16
        self._scale = self.head_dim ** -0.5
        self._lib = lib

    @classmethod
    def empty(cls, pages: int, page_tokens: int, heads: int, head_dim: int, storage: str = "bf16", device="cuda"):
        """A cache over new pages; storage "bf16", "f32" or "int4"."""
        torch = _torch()
        shape = (pages, heads, page_tokens)
        if storage == "int4":
            k, v = (torch.empty(shape + (head_dim // 2,), dtype=torch.uint8, device=device) for _ in range(2))
            groups = shape + (head_dim // AWA_CACHE_GROUP, 2)
            return cls(k, v, *(torch.empty(groups, dtype=torch.bfloat16, device=device) for _ in range(2)))
        dtype = {"bf16": torch.bfloat16, "f32": torch.float32}[storage]
        return cls(*(torch.empty(shape + (head_dim,), dtype=dtype, device=device) for _ in range(2)))

    def __del__(self):
        handle = getattr(self, "_handle", None)
        if handle and _lib is not None:
            _lib.awa_cache_destroy(handle)
            self._handle = None

    def _rows(self, batch: CacheBatch, t, name: str) -> int:
        """The token stride of a [rows, heads, head_dim] tensor of this batch."""
        shape, stride = t.shape, t.stride()
        if len(shape) != 3 or shape[0] != batch.rows or shape[2] != self.head_dim:
            raise ValueError(f"{name} must be [{batch.rows}, heads, {self.head_dim}]")
        if stride[2] != 1 or (stride[1] != shape[2] and shape[1] != 1):
            raise ValueError(f"{name} must be dense within a row")
        if t.device != self.device:
            raise ValueError(f"{name} is on {t.device}, the cache on {self.device}")
        # a single row's stride is never used, but has to hold a row
        return stride[0] if shape[0] > 1 else max(stride[0], shape[1] * shape[2])

    def _stream(self, batch: CacheBatch, stream):
        if batch.device != self.device:
            raise ValueError(f"the batch is on {batch.device}, the cache on {self.device}")
        if stream is not None:
            return stream.cuda_stream
        # a step of one row takes the GPU a few microseconds; the Stream object
        # that current_stream() builds would take the host two of its own
        return _current_raw_stream(self.device.index) if self.device.index is not None else None

    def _empty(self, shape, dtype, stream):
        """New memory that belongs to the stream the call runs on: what the
        allocator hands out may still be in use on any other."""
        torch = _torch()
        if stream is None:
            return torch.empty(shape, dtype=dtype, device=self.device)
        with torch.cuda.stream(stream):
            return torch.empty(shape, dtype=dtype, device=self.device)

    def _like(self, q, stream):
        if stream is None and q.is_contiguous():
            return _torch().empty_like(q)
        return q.new_empty(q.shape) if stream is None else self._empty(q.shape, q.dtype, stream)

    def append(self, batch: CacheBatch, k, v, q=None, rope: Optional[CacheRope] = None, q_out=None, stream=None):
        """Writes the batch's k (rotated) and v rows into the cache; returns q
        rotated (in q_out, by default a new tensor of q's type), None without q."""
        handle = self._stream(batch, stream)
        ks, vs = self._rows(batch, k, "k"), self._rows(batch, v, "v")
        if k.shape[1] != self.heads or v.shape[1] != self.heads:
            raise ValueError(f"k and v must have the cache's {self.heads} heads")
        if v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
            raise TypeError("q, k and v must share a dtype")
        if rope is not None:
            if rope.table.device != self.device:
                raise ValueError(f"the rope table is on {rope.table.device}, the cache on {self.device}")
            if rope.rows is not None and rope.rows != batch.rows:
                raise ValueError(f"coords must have {batch.rows} rows")
        heads, qp, qs, op, os_, ot = 0, None, 0, None, 0, AWA_BF16
        code = _dtype_code(k)
        if q is not None:
            heads, qp, qs = q.shape[1], q.data_ptr(), self._rows(batch, q, "q")
            if q_out is None:
                q_out, os_, ot = self._like(q, stream), heads * self.head_dim, code
            elif q_out.shape != q.shape:
                raise ValueError("q_out must have q's shape")
            else:
                os_, ot = self._rows(batch, q_out, "q_out"), _dtype_code(q_out)
            op = q_out.data_ptr()
        rc = self._lib.awa_cache_append(self._handle, batch.ref, heads, code, qp, qs, k.data_ptr(), ks, v.data_ptr(),
                                        vs, None if rope is None else rope.ref, ot, op, os_, handle)
        if rc:
            _check(rc)
        return q_out if q is not None else None

    def read(self, batch: CacheBatch, dtype=None, stream=None):
        """The batch's rows (k, v) [rows, heads, head_dim] back from the cache."""
        handle = self._stream(batch, stream)
        shape = (batch.rows, self.heads, self.head_dim)
        k, v = (self._empty(shape, dtype or self._rows_dtype, stream) for _ in range(2))
        row = self.heads * self.head_dim
        _check(self._lib.awa_cache_read(self._handle, batch.ref, _dtype_code(k), k.data_ptr(), row, v.data_ptr(), row,
                                        handle))
        return k, v

    def attention_workspace_bytes(self, batch: CacheBatch, q_heads: int, sinks: int = 0, window: int = 0,
                                  frame_tokens: int = 1) -> int:
        _check_mask(sinks, window, frame_tokens)
        return int(self._lib.awa_cache_attention_workspace_bytes(self._handle, batch.ref, q_heads, sinks, window,
                                                                 frame_tokens))

    def attention(self, batch: CacheBatch, q, sinks: int = 0, window: int = 0, frame_tokens: int = 1, scale=None,
                  out=None, workspace=None, stream=None):
        """softmax(scale q K^T) V of every row over the cached rows it sees (scale
        1 / sqrt(head_dim) by default): [rows, q_heads, head_dim]. A workspace
        given must not be in use by another call; one made here is not shared."""
        handle = self._stream(batch, stream)
        _check_mask(sinks, window, frame_tokens)
        if q.dtype != self._rows_dtype:
            raise TypeError(f"this cache takes {self._rows_dtype} rows")
        qs, heads = self._rows(batch, q, "q"), q.shape[1]
        if out is None:
            out, os_ = self._like(q, stream), heads * self.head_dim
        elif out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError("out must have q's shape and dtype")
        else:
            os_ = self._rows(batch, out, "out")
        space, need = None, 0
        if self.storage != AWA_F32:  # fp32 caches never need a workspace
            need = self._lib.awa_cache_attention_workspace_bytes(self._handle, batch.ref, heads, sinks, window,
                                                                 frame_tokens)
        if need:
            if workspace is None:
                workspace = self._empty(need, _torch().uint8, stream)
            elif workspace.device != self.device:
                raise ValueError(f"the workspace is on {workspace.device}, the cache on {self.device}")
            elif not workspace.is_contiguous():
                raise ValueError("the workspace must be contiguous")
            space, need = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        rc = self._lib.awa_cache_attention(self._handle, batch.ref, heads, self._type, q.data_ptr(), qs,
                                           self._scale if scale is None else scale, sinks, window, frame_tokens,
                                           out.data_ptr(), os_, space, need, handle)
        if rc:
            _check(rc)
        return out
