"""Attention of a chunk of new tokens over the cache, on the GPU, against the
formula in 64 bits over the values that the cache stores."""
from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from kvforge_b200 import FMT_F16, FMT_INT4, FMT_INT8, ORD_HEAD, ORD_TOKEN, api  # noqa: E402
from kvforge_b200.layout import Placement  # noqa: E402

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HEAD, TOKEN = Placement(ORD_HEAD, False, 0), Placement(ORD_TOKEN, False, 0)
HEAD16, TOKEN16, TOKEN128 = Placement(ORD_HEAD, True, 16), Placement(ORD_TOKEN, True, 16), Placement(ORD_TOKEN, True, 128)
FORMATS = [(FMT_F16, 0, 128), (FMT_INT8, 64, 128), (FMT_INT4, 32, 128), (FMT_F16, 0, 64), (FMT_INT8, 64, 64),
           (FMT_INT4, 64, 64), (FMT_INT8, 128, 128), (FMT_INT4, 128, 128)]


def _gen(cuda, seed):
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return g


def _randn(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=g.device).to(dtype)


def _cache(cuda, g, B, Hkv, n, d, fmt, group, place, seq_lens=None, loud=True):
    """A cache of normal keys and values, some channels eight times as large."""
    K, V = _randn((B, Hkv, n, d), g), _randn((B, Hkv, n, d), g)
    if loud:
        K[..., ::31] *= 8
        V[..., 5::37] *= 8
    c = api.KVCache.from_logical(K, V, fmt=fmt, group=group, place=place)
    if seq_lens is not None:
        c.seq_lens = torch.tensor(seq_lens, dtype=torch.int32, device=cuda)
    return c


def _values(cache):
    """Stored keys and values [B][n][Hkv][D] in 64 bits, whatever seq_lens says."""
    lens, cache.seq_lens = cache.seq_lens, None
    k, v = api.gather(cache, cache.n)
    cache.seq_lens = lens
    return k.double(), v.double()


def _exact(q, cache, q_lens, causal, scale=None):
    """(out, lse, tolerance) in 64 bits.

    Errors of the kernels: a score adds d products q k, each off by at most
    2^-21 relative (fp32 queries: two tf32 halves of each factor) or, for 16-bit
    queries over a quantized cache, by k's rounding to fp16 (2^-11); fp32
    accumulation of d terms and the scale add (d + 4) 2^-24. An error ds of
    every score moves each weight, and their sum, by a factor within 1 +- ds, so
    an output by at most 2 ds sum(p |v|); exp2f and the sums over tokens add
    (n + 16) 2^-24. For 16-bit queries weights and (quantized) values are
    rounded to fp16: 2^-11 each, and weights below fp16's normal range by 2^-25
    absolute of a row whose largest weight is 1. Then one rounding to the type."""
    B, T, H, d = q.shape
    k, v = _values(cache)
    scale = 1 / math.sqrt(d) if scale is None else scale
    n, Hkv, g = cache.n, cache.Hkv, H // cache.Hkv
    half = q.dtype != torch.float32
    quant = cache.fmt != FMT_F16
    out = torch.zeros((B, T, H, d), dtype=torch.float64, device=q.device)
    lse = torch.full((B, T, H), -math.inf, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    ql = [T] * B if q_lens is None else [min(max(x, 0), T) for x in q_lens]
    kv = [n] * B if cache.seq_lens is None else [min(max(x, 0), n) for x in cache.seq_lens.tolist()]
    for b in range(B):
        if ql[b] == 0 or kv[b] == 0:
            continue
        for h in range(H):
            kk, vv = k[b, : kv[b], h // g], v[b, : kv[b], h // g]
            qq = q[b, : ql[b], h].double()
            s = qq @ kk.T * scale
            last = kv[b] - ql[b] + torch.arange(ql[b], device=q.device) if causal else \
                torch.full((ql[b],), kv[b] - 1, device=q.device)
            hide = torch.arange(kv[b], device=q.device) > last[:, None]
            s.masked_fill_(hide, -math.inf)
            none = last < 0
            p = torch.softmax(s, -1).masked_fill(none[:, None], 0.0)
            out[b, : ql[b], h] = p @ vv
            lse[b, : ql[b], h] = torch.logsumexp(s, -1) * math.log2(math.e)
            mag = (qq.abs() @ kk.abs().T * abs(scale)).masked_fill(hide, 0.0).amax(-1, keepdim=True)
            ds = mag * ((2.0 ** -11 if half and quant else 2.0 ** -21) + (d + 4) * 2.0 ** -24)
            pv = p @ vv.abs()
            t = pv * (2 * ds * 1.01 + (n + 16) * 2.0 ** -24)
            if half:
                t = t + pv * (2.0 ** -11 + (2.0 ** -11 if quant else 0)) + \
                    2.0 ** -25 * p.amax(-1, keepdim=True) * vv.abs().sum(0)
            tol[b, : ql[b], h] = t
    tol = tol + (2.0 ** -24 if not half else torch.finfo(q.dtype).eps / 2) * (out.abs() + tol) + 2.0 ** -25
    return out, lse, tol


def _check(got, exact, what=""):
    out, _, tol = exact
    err = (got.double() - out).abs()
    assert bool((err <= tol).all()), f"{what}: off by {float((err / tol).max()):.3g} times the bound, nan {int(got.isnan().sum())}"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt,group,d", FORMATS)
@pytest.mark.parametrize("place", [HEAD, TOKEN, HEAD16, TOKEN128], ids=lambda p: p.name)
@pytest.mark.parametrize("causal", [True, False])
def test_formats_and_placements(cuda, dtype, fmt, group, d, place, causal):
    g = _gen(cuda, 1)
    B, T, H, Hkv, n = 2, 37, 6, 2, 205
    cache = _cache(cuda, g, B, Hkv, n, d, fmt, group, place, seq_lens=[205, 131])
    q = _randn((B, T, H, d), g, dtype)
    lse = torch.zeros((B, T, H), device=cuda)
    got = api.chunk_attention(q, cache, causal=causal, lse=lse)
    exact = _exact(q, cache, None, causal)
    _check(got, exact)
    assert float((lse.double() - exact[1]).abs().max()) < 2e-2
    assert api.device_errors() == 0


SHAPES = [
    # B, T, H, Hkv, n, seq_lens, q_lens
    (1, 1, 1, 1, 1, None, None),
    (1, 1, 8, 1, 1000, None, None),
    (3, 1, 7, 7, 333, [1, 0, 333], None),
    (2, 5, 5, 1, 64, [64, 3], [5, 5]),             # fewer stored than new: first rows see nothing
    (4, 9, 10, 5, 129, [129, 64, 0, 65], [9, 0, 4, 1]),
    (2, 63, 16, 2, 128, None, [63, 64]),           # 64 counts as T
    (1, 128, 4, 4, 128, None, None),               # a whole prompt
    (1, 300, 14, 2, 700, [650], [257]),
    (2, 130, 40, 5, 2000, [1999, 1500], [130, 77]),
    (1, 3, 64, 4, 4097, None, None),
    (1, 257, 2, 1, 513, None, None),
    (5, 2, 12, 1, 100, [-3, 1, 2, 500, 99], [2, 2, 2, 2, -1]),  # lengths outside their range
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt,group,d", [(FMT_F16, 0, 128), (FMT_INT8, 64, 128), (FMT_INT4, 32, 64)])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:5])))
@pytest.mark.parametrize("causal", [True, False])
def test_shapes_and_lengths(cuda, dtype, fmt, group, d, shape, causal):
    B, T, H, Hkv, n, seq_lens, q_lens = shape
    g = _gen(cuda, 2)
    cache = _cache(cuda, g, B, Hkv, n, d, fmt, group, TOKEN16, seq_lens=seq_lens)
    q = _randn((B, T, H, d), g, dtype)
    exact = _exact(q, cache, q_lens, causal)
    dlens = None if q_lens is None else torch.tensor(q_lens, dtype=torch.int32, device=cuda)
    for splits in (1, None, 7):
        out = torch.full_like(q, 7.0)
        lse = torch.full((B, T, H), 7.0, device=cuda)
        ws = api.ChunkWorkspace.allocate(cache, T, H, dtype, splits=splits)
        for x in (ws.part_o, ws.part_ml):
            if x is not None:
                x.fill_(float("nan"))  # whatever an earlier call left there
        api.chunk_attention(q, cache, q_lens=dlens, causal=causal, out=out, lse=lse, workspace=ws)
        assert api.device_errors() == 0
        for b in range(B):
            m = T if q_lens is None else min(max(q_lens[b], 0), T)
            assert bool((out[b, m:] == 7.0).all()) and bool((lse[b, m:] == 7.0).all())
            _check(out[b, :m], tuple(x[b, :m] for x in exact), f"sequence {b}, splits {splits}")
            none = exact[1][b, :m] == -math.inf
            assert bool((lse[b, :m][none] == -math.inf).all()) and not out[b, :m][none].any()
            assert bool(((lse[b, :m] - exact[1][b, :m])[~none].abs() < 2e-2).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_what_a_row_does_not_see_has_no_effect(cuda, dtype, d):
    """Infinities, NaN and huge values at tokens past the end and past each
    causal row, and in pages that no block maps: the rows before them are
    those of a cache that holds zeros there."""
    g = _gen(cuda, 3)
    B, T, H, Hkv, n = 2, 70, 4, 2, 400
    for place in (TOKEN16, HEAD):
        cache = _cache(cuda, g, B, Hkv, n, d, FMT_F16, 0, place, seq_lens=[390, 201])
        K, V = (x.float().transpose(1, 2).contiguous() for x in _values(cache))
        K2, V2 = K.clone(), V.clone()
        for b, kv in ((0, 390), (1, 201)):
            K2[b, :, kv:], V2[b, :, kv:] = float("nan"), float("inf")
            K[b, :, kv:], V[b, :, kv:] = 0, 0
            # the last token's own row: seen by the last query alone
            V2[b, 0, kv - 1, 3], V2[b, 1, kv - 1, 7], K2[b, 1, kv - 1, 1] = float("inf"), float("nan"), float("nan")
            V2[b, 0, kv - 31, 9] = float("-inf")
        a = api.KVCache.from_logical(K, V, fmt=FMT_F16, place=place)
        c = api.KVCache.from_logical(K2, V2, fmt=FMT_F16, place=place)
        a.seq_lens = c.seq_lens = cache.seq_lens
        q = _randn((B, T, H, d), g, dtype)
        exact = _exact(q, a, None, True)
        for splits in (1, 3):
            ws = api.ChunkWorkspace.allocate(a, T, H, dtype, splits=splits)
            x, y = (api.chunk_attention(q, z, workspace=ws) for z in (a, c))
            # a step that holds an infinity may add in another order; the bound of _exact holds for any
            _check(y[:, : T - 31], tuple(e[:, : T - 31] for e in exact))
            assert not x.isnan().any() and not x.isinf().any()
            # rows T - 31 .. T - 2 see one infinity, in one column of KV head 0
            cols = torch.ones(d, dtype=torch.bool, device=cuda)
            cols[9] = False
            late, late_y = x[:, T - 31: T - 1], y[:, T - 31: T - 1]
            assert not late_y[:, :, :2, 9].isfinite().any()  # infinity, or NaN where its weight rounds to 0
            tol = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -9  # another order of the same sums
            assert bool(((late - late_y)[..., cols].abs() <= tol * (late[..., cols].abs() + 1)).all())
            assert bool(((late - late_y)[:, :, 2:, 9].abs() <= tol * (late[:, :, 2:, 9].abs() + 1)).all())
            # the last row: infinity in column 3, NaN in column 7 or, by a NaN key, everywhere
            assert not y[:, T - 1, :2, 3].isfinite().any() and bool(y[:, T - 1, 2:].isnan().all())
    assert api.device_errors() == 0


def test_bad_pages_count_as_zero(cuda):
    g = _gen(cuda, 4)
    B, T, H, Hkv, n, d = 1, 4, 2, 1, 64, 128
    cache = _cache(cuda, g, B, Hkv, n, d, FMT_INT8, 64, TOKEN16)
    cache.block_table[0, 1] = -1
    q = _randn((B, T, H, d), g, torch.bfloat16)
    k, v = api.gather(cache, n)
    assert api.device_errors() == 4
    full = api.KVCache.from_logical(k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous(), fmt=FMT_F16, place=TOKEN)
    a, b = api.chunk_attention(q.float(), cache), api.chunk_attention(q.float(), full)
    assert float((a - b).abs().max()) < 2e-2  # the second cache rounds the values to fp16
    assert api.chunk_attention(q, cache).isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_scale_and_large_scores(cuda, dtype):
    g = _gen(cuda, 5)
    B, T, H, Hkv, n, d = 2, 21, 6, 3, 150, 128
    cache = _cache(cuda, g, B, Hkv, n, d, FMT_F16, 0, TOKEN)
    for off in (0, 8, 1):  # the last one off 16-byte boundaries
        big = _randn((T, B, (H + 6) * d + off), g, dtype)
        q = big[..., off: off + H * d].unflatten(-1, (H, d)).transpose(0, 1)
        buf = torch.zeros((T, B, H * d + 9), dtype=dtype, device=cuda)
        out = buf[..., off: off + H * d].unflatten(-1, (H, d)).transpose(0, 1)
        api.chunk_attention(q, cache, out=out, scale=0.3)
        _check(out, _exact(q, cache, None, True, scale=0.3))
        assert not buf[..., :off].any() and not buf[..., off + H * d:].any()
    # scores in the thousands: one token takes all, the sums must not overflow
    for mul in (100.0, 1e-6):
        q = (_randn((B, T, H, d), g) * mul).to(dtype)
        got = api.chunk_attention(q, cache)
        assert got.isfinite().all()
        if mul < 1 or dtype == torch.float32:
            continue
        top = _exact(q, cache, None, True)[0]
        assert float((got.double() - top).abs().max()) < 0.2
    if dtype == torch.bfloat16:  # queries past fp16's range, and far below it
        q = _randn((B, T, H, d), g) * 1e6
        a = api.chunk_attention(q.to(dtype), cache, scale=1e-7)
        _check(a, _exact(q.to(dtype), cache, None, True, scale=1e-7))
        q = _randn((B, T, H, d), g) * 1e-9
        a = api.chunk_attention(q.to(dtype), cache, scale=1e8)
        _check(a, _exact(q.to(dtype), cache, None, True, scale=1e8))


def test_a_growing_maximum(cuda):
    """Scores that rise along the sequence: every step raises the running maximum."""
    g = _gen(cuda, 6)
    B, T, H, Hkv, n, d = 1, 33, 2, 1, 1500, 128
    K = torch.zeros((B, Hkv, n, d), device=cuda)
    K[..., 0] = torch.arange(n, device=cuda) / 8
    V = _randn((B, Hkv, n, d), g)
    cache = api.KVCache.from_logical(K, V, fmt=FMT_F16, place=TOKEN)
    for dtype in DTYPES:
        q = torch.zeros((B, T, H, d), dtype=dtype, device=cuda)
        q[..., 0, 0], q[..., 1, 0] = 2.0, -2.0  # rising and falling
        for splits in (1, 4):
            ws = api.ChunkWorkspace.allocate(cache, T, H, dtype, splits=splits)
            _check(api.chunk_attention(q, cache, workspace=ws), _exact(q, cache, None, True), f"{dtype}")


def test_one_token_is_a_decode_step(cuda):
    g = _gen(cuda, 7)
    B, H, Hkv, n, d = 4, 16, 4, 900, 128
    lens = [900, 1, 333, 0]
    for fmt, group in ((FMT_F16, 0), (FMT_INT8, 64), (FMT_INT4, 32)):
        cache = _cache(cuda, g, B, Hkv, n, d, fmt, group, TOKEN16, seq_lens=lens)
        q = _randn((B, H, d), g)
        a = api.decode(q, cache)
        b = api.chunk_attention(q[:, None], cache)[:, 0]
        assert float((a - b).abs().max()) < 1e-4


def test_repeats_streams_and_graphs(cuda):
    """The same call gives the same bits, on a side stream and replayed from a graph that reads new inputs."""
    g = _gen(cuda, 8)
    B, T, H, Hkv, n, d = 2, 40, 8, 2, 1200, 128
    for dtype in (torch.float32, torch.bfloat16):
        cache = _cache(cuda, g, B, Hkv, n, d, FMT_INT8, 64, TOKEN16, seq_lens=[1200, 700])
        q = _randn((B, T, H, d), g, dtype)
        first = api.chunk_attention(q, cache)
        assert torch.equal(first, api.chunk_attention(q, cache))
        side = torch.cuda.Stream(cuda)
        side.wait_stream(torch.cuda.current_stream(cuda))
        x = api.chunk_attention(q, cache, stream=side)
        side.synchronize()
        assert torch.equal(x, first)
        ws = api.ChunkWorkspace.allocate(cache, T, H, dtype)
        out = torch.zeros_like(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            api.chunk_attention(q, cache, out=out, workspace=ws)
        for lens in ([1200, 700], [40, 1100], [0, 13]):
            q.copy_(_randn(q.shape, g, dtype))
            cache.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
            out.zero_()
            graph.replay()
            _check(out, _exact(q, cache, None, True), f"lengths {lens}")
    assert api.device_errors() == 0


@pytest.mark.parametrize("fmt,group,place", [(FMT_INT8, 64, TOKEN16), (FMT_INT4, 32, HEAD), (FMT_F16, 0, HEAD16)])
def test_prompt_in_chunks_then_decode(cuda, fmt, group, place):
    """A prompt in chunks of unequal lengths through append_rope and
    chunk_attention, then decode steps, as they are used together: every output
    is that of the whole cache, and equals one call over the whole prompt."""
    g = _gen(cuda, 9)
    B, H, Hkv, n, d = 2, 8, 2, 256, 128
    z = torch.zeros((B, Hkv, n, d), device=cuda)
    cache = api.KVCache.from_logical(z, z, fmt=fmt, group=group, place=place)
    cache.seq_lens = torch.zeros(B, dtype=torch.int32, device=cuda)
    rope = api.Rope.build(n, d, device=cuda)
    w = 1 + 0.1 * _randn((d,), g)
    done = [0, 0]
    for T, lens in ((100, [100, 60]), (1, [1, 1]), (70, [3, 70]), (4, [4, 4])):
        qkv = _randn((B, T, H + 2 * Hkv, d), g, torch.bfloat16)
        q, k, v = qkv.split((H, Hkv, Hkv), 2)
        dl = torch.tensor(lens, dtype=torch.int32, device=cuda)
        q = api.append_rope(cache, k, v, rope, lens=dl, k_weight=w, q=q, q_weight=w)
        done = [x + y for x, y in zip(done, lens)]
        assert cache.seq_lens.tolist() == done
        out = api.chunk_attention(q, cache, q_lens=dl)
        exact = _exact(q, cache, lens, True)
        for b, m in enumerate(lens):
            _check(out[b, :m], tuple(x[b, :m] for x in exact), f"chunk of {T}")
    for _ in range(2):
        qkv = _randn((B, 1, H + 2 * Hkv, d), g, torch.float32)
        q, k, v = qkv.split((H, Hkv, Hkv), 2)
        q = api.append_rope(cache, k, v, rope, k_weight=w, q=q, q_weight=w)
        step = api.decode(q[:, 0].contiguous(), cache)
        assert float((step - api.chunk_attention(q, cache)[:, 0]).abs().max()) < 1e-4
    assert api.device_errors() == 0


def test_refusals(cuda):
    g = _gen(cuda, 10)
    cache = _cache(cuda, g, 2, 2, 32, 64, FMT_F16, 0, TOKEN)
    q = _randn((2, 3, 4, 64), g)
    lens = torch.tensor([1, 2], dtype=torch.int32, device=cuda)
    for f in (lambda: api.chunk_attention(q[:1], cache), lambda: api.chunk_attention(q[:, :, :3], cache),
              lambda: api.chunk_attention(q[..., :32], cache), lambda: api.chunk_attention(q.double(), cache),
              lambda: api.chunk_attention(q.transpose(2, 3), cache), lambda: api.chunk_attention(q[:, :, :0], cache),
              lambda: api.chunk_attention(q, cache, q_lens=lens.long()), lambda: api.chunk_attention(q, cache, q_lens=lens[:1]),
              lambda: api.chunk_attention(q, cache, out=q.half()), lambda: api.chunk_attention(q, cache, out=q[:, :2]),
              lambda: api.chunk_attention(q, cache, lse=torch.zeros(3, device=cuda)),
              lambda: api.chunk_attention(q.cpu(), cache),
              lambda: api.chunk_attention(q, cache, workspace=api.ChunkWorkspace.allocate(cache, 2, 4, q.dtype, splits=2))):
        with pytest.raises(ValueError):
            f()
    assert api.chunk_attention(q[:, :0], cache).numel() == 0
    assert api.device_errors() == 0


@pytest.mark.parametrize("fmt,group,d", [(FMT_F16, 0, 128), (FMT_F16, 0, 64), (FMT_INT8, 64, 128), (FMT_INT4, 32, 128)])
def test_few_rows_over_many_steps(cuda, fmt, group, d):
    """One row tile taken in turn by both softmax groups, who share its queries: the
    group that ends first must not disturb the other (uneven numbers of steps,
    repeated, on every SM at once)."""
    g = _gen(cuda, 11)
    B, T, H, Hkv = 40, 4, 32, 4
    for n in (1, 128, 129, 640, 1153):
        cache = _cache(cuda, g, B, Hkv, n, d, fmt, group, TOKEN16)
        q = _randn((B, T, H, d), g, torch.bfloat16)
        exact = _exact(q, cache, None, True)
        ws = api.ChunkWorkspace.allocate(cache, T, H, q.dtype, splits=2)
        first = api.chunk_attention(q, cache, workspace=ws)
        _check(first, exact, f"n = {n}")
        for _ in range(20):
            assert torch.equal(api.chunk_attention(q, cache, workspace=ws), first)
    assert api.device_errors() == 0
