"""kvf_b200_chunk_splits: splits where they pay, and never without a bound."""
from __future__ import annotations

import pytest

from kvforge_b200._native import DT_BF16, DT_F32, FMT_F16, FMT_INT8, lib


def splits(B, T, H, Hkv, n, fmt=FMT_INT8, d=128, dtype=DT_BF16):
    return lib().kvf_b200_chunk_splits(B, T, H, Hkv, n, fmt, d, dtype)


@pytest.mark.parametrize("shape", [(64, 512, 64, 8, 131072), (64, 512, 64, 8, 65536), (1, 32768, 64, 64, 131072),
                                   (1, 32768, 64, 8, 131072), (512, 16, 64, 8, 1024), (4096, 16, 64, 8, 1024)])
def test_large_batches_stay_whole(shape):
    """Enough blocks for many waves: what splitting rounds off is less than its partials cost."""
    assert splits(*shape) == 1


@pytest.mark.parametrize("shape,least", [((64, 4, 64, 8, 16384), 2), ((1, 4096, 32, 8, 32768), 2), ((1, 1, 32, 8, 131072), 16),
                                         ((1, 2048, 32, 8, 131072), 2)])
def test_few_blocks_are_split(shape, least):
    assert splits(*shape) >= least


def test_partials_are_bounded():
    for dtype in (DT_BF16, DT_F32):
        for fmt in (FMT_F16, FMT_INT8):
            for d in (64, 128):
                for B in (1, 3, 16, 100, 1000, 10000):
                    for T in (1, 3, 16, 100, 1000, 10000):
                        for H, Hkv in ((8, 8), (8, 1), (64, 8), (40, 5)):
                            for n in (1, 100, 1000, 32768, 1 << 20):
                                s = splits(B, T, H, Hkv, n, fmt, d, dtype)
                                assert s >= 1 and (s == 1 or B * T * H * s * (d + 2) * 4 <= 512 << 20)
