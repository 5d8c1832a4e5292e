"""Argument checks of the MXFP4 and drafted-tree calls that need no GPU."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch


def test_null_contexts_are_rejected(wrs):
    lib = wrs._lib.lib()
    f = np.zeros(64, np.float32)
    p = f.ctypes.data_as(ctypes.c_void_p)
    one = (ctypes.c_size_t * 1)(0)
    ptrs = (ctypes.c_void_p * 1)(f.ctypes.data)
    assert lib.wrs_attn_tree_self(None, None, 0, one, one, 1, p, 1, p, 64, p, 64) == -1
    assert lib.wrs_kv_keep_rows(None, one, one, 1, one, 1) == -1
    assert lib.wrs_mx4_quantize(None, 0, p, 64, 64, 1, 64, p, 32, p, 2) == -1
    assert lib.wrs_mx4_dequantize(None, p, 32, p, 2, 1, 64, 0, p, 64, 64) == -1
    assert lib.wrs_linear_mx4(None, 0, p, None, 64, 64, 1, ptrs, ptrs, None, 1, 64, 1, 0, 0, ptrs,
                              one, 1, 64) == -1


def test_mx4_holds_matching_rows(wrs):
    m = wrs.Mx4.empty(3, 96, device="cpu")
    assert m.shape == (3, 96) and m.codes.shape == (3, 48) and m.scales.shape == (3, 3)
    with pytest.raises(AssertionError):
        wrs.Mx4.empty(3, 40, device="cpu")
    with pytest.raises(AssertionError):
        wrs.Mx4(torch.zeros((3, 48), dtype=torch.uint8), torch.zeros((3, 4), dtype=torch.uint8))
    with pytest.raises(AssertionError):
        wrs.Mx4(torch.zeros((2, 48), dtype=torch.uint8), torch.zeros((3, 3), dtype=torch.uint8))
    with pytest.raises(TypeError):
        wrs.Mx4(torch.zeros((3, 48)), torch.zeros((3, 3), dtype=torch.uint8))
    with pytest.raises(TypeError):
        wrs.Mx4(torch.zeros((3, 96), dtype=torch.uint8)[:, ::2],
                torch.zeros((3, 3), dtype=torch.uint8))
