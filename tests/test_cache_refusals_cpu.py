"""What the small cache's operators decide on the host, before anything touches a device."""

import ctypes

import torch

from attention_b200 import _lib, int4


def test_compaction_refuses_pools_that_share_memory():
    """Each pool is moved by clusters of its own: the same memory twice would be moved twice."""
    lay = _lib.KvLayout(None, None, 64, 0, 16, 8, 4096, 4, 8)  # 64 rows; never dereferenced
    for second in (1 << 20, (1 << 20) + 64 * 128 - 16, (1 << 20) - 64 * 32 + 16):
        ptrs, sizes = (ctypes.c_void_p * 2)(1 << 20, second), (ctypes.c_int * 2)(128, 32)
        assert _lib.lib.spa_compact_tokens(ctypes.byref(lay), 2, ptrs, sizes, 1, 2, 4096, 4, None, 0,
                                           None) == _lib.SPA_ERR_INVALID


def test_workspace_sizes_are_those_of_the_tensors_device(monkeypatch):
    """On a machine of unlike GPUs a size asked for one is not given to another, whichever is current."""
    current, sms = [0], {0: 148, 1: 132}

    class On:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            self.before, current[0] = current[0], self.device

        def __exit__(self, *_):
            current[0] = self.before

    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(int4._lib, "lib", type("Lib", (), {
        "spa_cache_decode_workspace_size": staticmethod(lambda *shape: sms[current[0]] * sum(shape))}))
    int4.cache_decode_workspace.cache_clear()
    try:
        shape = (1, 8, 8, 64, 4096, 4096, 0, -1)
        for _ in range(2):
            assert [int4.cache_decode_workspace(d, *shape) for d in (0, 1)] == [sms[d] * sum(shape) for d in (0, 1)]
    finally:
        int4.cache_decode_workspace.cache_clear()
