"""Argument checks of the long-session calls that need no GPU."""
from __future__ import annotations

import ctypes

import numpy as np


def test_null_handles_are_rejected(wrs):
    lib = wrs._lib.lib()
    f = np.zeros(64, np.float32)
    p = f.ctypes.data_as(ctypes.c_void_p)
    one = (ctypes.c_size_t * 1)(0)
    assert lib.wrs_kv_append_rows(None, 0, one, one, 1, p, 64, 64, p, 64, 64) == -1
    assert lib.wrs_kv_read_rows(None, 0, one, one, one, 1, p, 64, 64, p, 64, 64) == -1
    assert lib.wrs_kv_read_cross(None, 0, 0, 1, p, 64, 64, p, 64, 64) == -1
    assert lib.wrs_attn_window_self(None, None, 0, one, one, 1, 1, 0, p, 64, 64, p, 64, 64) == -1
    assert lib.wrs_token_logprobs(None, 0, p, 64, 64, 1, 64, None, 0, 0, 1.0, None, None, p, 0,
                                  None, None) == -1


def test_the_package_offers_them(wrs):
    assert "token_logprobs" in wrs.__all__ and callable(wrs.token_logprobs)
    assert wrs.WRS_I8 == 4
    for name in ("append_rows", "read_rows", "read_cross", "window_self"):
        assert callable(getattr(wrs.KvArena, name))
