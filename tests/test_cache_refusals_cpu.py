"""Calls of the small cache's operators that are refused before anything touches the device."""

import ctypes

from attention_b200 import _lib


def test_compaction_refuses_pools_that_share_memory():
    """Each pool is moved by clusters of its own: the same memory twice would be moved twice."""
    lay = _lib.KvLayout(None, None, 64, 0, 16, 8, 4096, 4, 8)  # 64 rows; never dereferenced
    for second in (1 << 20, (1 << 20) + 64 * 128 - 16, (1 << 20) - 64 * 32 + 16):
        ptrs, sizes = (ctypes.c_void_p * 2)(1 << 20, second), (ctypes.c_int * 2)(128, 32)
        assert _lib.lib.spa_compact_tokens(ctypes.byref(lay), 2, ptrs, sizes, 1, 2, 4096, 4, None, 0,
                                           None) == _lib.SPA_ERR_INVALID
