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
@pytest.mark.parametrize("far", [17.0, 18.0])
@pytest.mark.parametrize("sink", [0, 20000, -1])
def test_many_small_weights_beside_a_large_one(cuda, dtype, far, sink):
    """One token takes nearly all of the softmax and its value is zero; 32768
    others, each e^-far of it, make the output.

    Bound: fp16 weights are taken against a largest one of at least 2^7 (a row's
    reference lies 7 below its maximum), and below fp16's normal range they are off by at most
    2^-25 absolute, 2^-32 of the largest; above it by 2^-11 relative. fp32
    queries: 2^-20 relative, from the products' and scores' halves. Scores are
    one product with 1, exact; exponentials, sums over n tokens and the merge
    add (n + 32) 2^-24 relative, and the output is rounded once."""
    g = _gen(cuda, 1)
    n, d, T, H = 32769, 128, 2, 2
    K = torch.zeros((1, 1, n, d), device=cuda)
    K[..., 0] = -far + _randn((1, 1, n), g) / 8
    K[0, 0, sink, 0] = 0
    V = _randn((1, 1, n, d), g) + 1
    V[0, 0, sink] = 0
    cache = api.KVCache.from_logical(K, V, fmt=FMT_F16, place=TOKEN)
    q = torch.zeros((1, T, H, d), dtype=dtype, device=cuda)
    q[..., 0] = 1
    k, v = (x[0, :, 0].double() for x in api.gather(cache, n))
    w = (k[:, 0]).exp()
    out = (w @ v) / w.sum()
    small = 2.0 ** -32 * v.abs().sum(0) / w.sum() if dtype != torch.float32 else 0.0
    rel = (2.0 ** -11 if dtype != torch.float32 else 2.0 ** -20) + (n + 32) * 2.0 ** -24
    tol = small + rel * (w @ v.abs()) / w.sum()
    tol = tol + torch.finfo(dtype).eps / 2 * (out.abs() + tol)
    for splits in (1, 2, 5):
        got = _attend(q, cache, splits, causal=False, scale=1.0).double()
        err = (got - out).abs()
        assert bool((err <= tol).all()), f"splits {splits}: off by {float((err / tol).max()):.3g} times the bound, " \
                                         f"{float((err / out.abs()).median()):.3g} relative"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e9, 1e35])
def test_scores_far_past_the_usual_range(cuda, dtype, size):
    """Scores of 1e5 to 1e36: the softmax is the token with the largest score, or
    the mean of the values of tokens whose keys are equal. fp16 queries reach
    as far as their type allows, against large keys."""
    g = _gen(cuda, 2)
    B, T, H, Hkv, n, d = 2, 70, 4, 2, 300, 128
    K, V = _randn((B, Hkv, n, d), g), _randn((B, Hkv, n, d), g)
    q = _randn((B, T, H, d), g)
    if dtype == torch.float16:
        K *= 4e3 if size > 1e20 else 30.0  # three times a key of this size is still below 65504
        q *= 1e4 if size > 1e20 else 3e3
    else:
        q *= size
    for b in range(B):  # equal keys in other halves of a step, and in other steps
        K[b, :, 5], K[b, :, 100], K[b, :, 201] = 3 * K[b, :, 40], 3 * K[b, :, 40], 3 * K[b, :, 40]
    cache = api.KVCache.from_logical(K, V, fmt=FMT_F16, place=TOKEN16)
    k, v = (x.double() for x in api.gather(cache, n))
    q = q.to(dtype)
    g2 = H // Hkv
    seen_gap = 0
    for splits in (1, 2, 3):
        lse = torch.zeros((B, T, H), device=cuda)
        got = _attend(q, cache, splits, lse=lse)
        assert bool(got.isfinite().all()) and bool(lse.isfinite().all()), f"splits {splits}"
        for b in range(B):
            for h in range(H):
                s = q[b, :, h].double() @ k[b, :, h // g2].T / math.sqrt(d)
                last = n - T + torch.arange(T, device=cuda)
                s.masked_fill_(torch.arange(n, device=cuda) > last[:, None], -math.inf)
                p = torch.softmax(s, -1)
                # fp32 scores are off by at most (d + 4) 2^-24 + 2^-21 of what they add; rows whose
                # runner-up is nearer than that (and 30 for the weights) have no answer in fp32
                mag = (q[b, :, h].double().abs() @ k[b, :, h // g2].abs().T / math.sqrt(d)).amax(-1)
                top = s.amax(-1)
                rest = torch.where(s == top[:, None], -math.inf, s).amax(-1)
                clear = top - rest > 2 * mag * ((d + 4) * 2.0 ** -24 + 2.0 ** -21) + 30
                seen_gap += int(clear.sum())
                err = (got[b, :, h].double() - p @ v[b, :, h // g2]).abs()[clear]
                tol = (2.0 ** -18 if dtype == torch.float32 else 2.0 ** -10 + torch.finfo(dtype).eps) * 5
                assert bool((err <= tol).all()), f"splits {splits}: {float(err.max()):.3g}"
                want = top * math.log2(math.e)
                assert bool(((lse[b, :, h].double() - want).abs()[clear] <= 1 + 1e-4 * want.abs()[clear]).all())
    assert seen_gap > 3 * B * T * H // 2  # most rows are clear


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
