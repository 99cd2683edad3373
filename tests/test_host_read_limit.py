"""Lengths that read_kv refuses, before any CUDA call."""
import ctypes as C

import pytest
import torch

import jaxmodules_b200 as jm
from jaxmodules_b200 import _native as nat


@pytest.mark.parametrize("L", [2**31 - 1, 2**31 - 16, 2**31 - 4096])
def test_lengths_that_would_not_fit_when_rounded_up(L):
    """(with 32 sequences the number of CTAs came out as 32, and the call as done)"""
    c = nat.PagedCacheArgs(k=16, v=16, page_table=16, pages=1, page_size=1, Hkv=1, d=8, B=32, width=1, dtype=nat.BMA_DTYPE_BF16)
    k = nat.Tensor(ptr=16, dtype=nat.BMA_DTYPE_BF16)
    assert nat.lib().bma_read_kv(C.byref(c), C.c_void_p(16), L, C.byref(k), C.byref(k), None) == nat.BMA_ERR_LIMIT
    with pytest.raises(ValueError, match="max_length"):
        jm.read_kv(jm.PagedCache.empty(1, 1, 1, 8, torch.zeros((1, 1), dtype=torch.int32)), torch.zeros(1, dtype=torch.int32), L)
