"""Attention of a chunk over the cache at the ends of its range, on the GPU:
infinities in the cache, weights far below the row's largest, scores far past
fp16's and fp32's usual range, NaN queries, metadata on odd words."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from kvforge_b200 import FMT_F16, FMT_INT4, FMT_INT8, ORD_HEAD, ORD_TOKEN, api  # noqa: E402
from kvforge_b200.layout import Placement  # noqa: E402

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HEAD, TOKEN, TOKEN16 = Placement(ORD_HEAD, False, 0), Placement(ORD_TOKEN, False, 0), Placement(ORD_TOKEN, True, 16)


def _gen(cuda, seed):
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return g


def _randn(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=g.device).to(dtype)


def _attend(q, cache, splits, lse=None, **kw):
    ws = api.ChunkWorkspace.allocate(cache, q.shape[1], q.shape[2], q.dtype, splits=splits)
    return api.chunk_attention(q, cache, workspace=ws, lse=lse, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt,group", [(FMT_F16, 0), (FMT_INT8, 64)])
@pytest.mark.parametrize("rows", [5, 90])
def test_rows_do_not_depend_on_their_neighbours(cuda, dtype, fmt, group, rows):
    """A row's output and lse are the same bits whatever queries stand beside it."""
    g = _gen(cuda, 7)
    B, T, H, Hkv, n, d = 2, rows, 6, 2, 700, 128
    cache = api.KVCache.from_logical(_randn((B, Hkv, n, d), g), _randn((B, Hkv, n, d), g), fmt=fmt, group=group, place=TOKEN16)
    q = _randn((B, T, H, d), g, dtype)
    other = torch.rand((B, T, H), generator=g, device=cuda) < 0.5
    for splits in (1, 2, 3):
        lse, lse2 = torch.zeros((2, B, T, H), device=cuda)
        x = _attend(q, cache, splits, lse=lse)
        for mul in (5.0, 0.0, math.nan):
            y = _attend(torch.where(other[..., None], q * mul, q), cache, splits, lse=lse2)
            assert torch.equal(x[~other], y[~other]) and torch.equal(lse[~other], lse2[~other])
    assert api.device_errors() == 0
