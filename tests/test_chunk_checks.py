"""kvf_b200_chunk_attention's alignment rules, checked before anything touches a GPU."""
from __future__ import annotations

import ctypes

import pytest

from kvforge_b200._native import DT_BF16, DT_F16, KvfArgs, KvfHeads, lib

FAKE = 0x1000  # never dereferenced: every call fails before a launch
MISALIGNED = 716


@pytest.mark.parametrize("dtype", [DT_F16, DT_BF16])
@pytest.mark.parametrize("fmt,shift,off", [(1, 6, 4), (2, 5, 8), (2, 5, 4), (2, 6, 4)])
@pytest.mark.parametrize("name", ["k_meta", "v_meta"])
def test_metadata_of_16_bit_queries_is_aligned_to_a_row(dtype, fmt, shift, off, name):
    a = KvfArgs()
    a.k = a.v = a.k_meta = a.v_meta = FAKE
    a.B, a.H, a.Hkv, a.n, a.group_shift, a.splits = 2, 8, 8, 64, shift, 1
    setattr(a, name, FAKE + off)
    q = KvfHeads(p=FAKE, dtype=dtype, heads=8, stride_b=1024, stride_t=1024, stride_h=128)
    assert lib().kvf_b200_chunk_attention(ctypes.byref(a), fmt, 128, 1, 0, ctypes.byref(q), ctypes.byref(q), 3, None, 1,
                                          None) == MISALIGNED
