"""The paged key/value cache on a B200: calls that its documentation allows and
that come near an edge (memory, magnitudes, sizes, masks)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import awa_b200
from awa_b200 import cache as binding

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- the memory
def create(k, v, pages=4):
    handle = ctypes.c_void_p()
    params = binding._CacheParams(awa_b200.AWA_BF16, 2, 64, 16, pages, k, v, 2 * 16 * 64, 16 * 64, None, None, 0, 0)
    lib = binding._cache_library()
    rc = lib.awa_cache_create(ctypes.byref(params), ctypes.byref(handle))
    if handle.value:
        lib.awa_cache_destroy(handle)
    return rc, lib.awa_last_error().decode()


def test_memory_that_the_gpu_cannot_reach_is_refused():
    """Refused when the handle is made: no kernel runs."""
    on_gpu = torch.empty(4, 2, 16, 64, dtype=torch.bfloat16, device="cuda")
    on_host = torch.empty(4, 2, 16, 64, dtype=torch.bfloat16)
    pointer = (on_host.data_ptr() + 15) // 16 * 16
    assert create(on_gpu.data_ptr(), on_gpu.data_ptr())[0] == awa_b200.AWA_OK
    for k, v in ((pointer, on_gpu.data_ptr()), (on_gpu.data_ptr(), pointer)):
        rc, error = create(k, v)
        assert rc == awa_b200.AWA_ERR_INVALID and "GPU" in error
