"""The calls around the cache where they meet its ends, on the GPU."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from kvforge_b200 import FMT_F16, FMT_INT4, FMT_INT8, ORD_HEAD, ORD_TOKEN, api  # noqa: E402
from kvforge_b200.layout import Placement  # noqa: E402

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
FORMATS = [(FMT_F16, 0), (FMT_INT8, 64), (FMT_INT4, 32)]


def _gen(cuda, seed):
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return g


def _randn(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=g.device).to(dtype)


@pytest.mark.parametrize("fmt,group", FORMATS)
def test_decode_of_blocks_without_a_page_stays_in_the_cache(cuda, fmt, group):
    """Lengths past the mapped blocks (an append that was reported, whose error
    nobody looked at): decode reads page 0 there, finite values, and sequences
    whose blocks are mapped are those of a cache that is right."""
    g = _gen(cuda, 4)
    B, H, Hkv, n, d = 8, 32, 4, 600, 128
    lens = [300, 599, 600, 17, 128, 600, 1, 256]
    K, V = _randn((B, Hkv, n, d), g), _randn((B, Hkv, n, d), g)
    q = _randn((B, H, d), g)
    for order in (ORD_HEAD, ORD_TOKEN):
        cache = api.KVCache.from_logical(K, V, fmt=fmt, group=group, place=Placement(order, True, 16), seq_lens=lens)
        want = api.decode(q, cache)
        cache.seq_lens[3] = cache.seq_lens[6] = 600
        for path in ("auto", "mma") + (("tc",) if fmt == FMT_INT8 else ()):
            got = api.decode(q, cache, path=path)
            assert bool(got.isfinite().all())
            rest = [0, 1, 2, 4, 5, 7]
            assert float((got[rest] - want[rest]).abs().max()) < 1e-4
        assert api.device_errors() == 0
