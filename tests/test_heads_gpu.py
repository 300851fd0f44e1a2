"""Norm and rotation of head vectors, the rotated append and the cache read
back, on the GPU, against the formulas in 64 bits and, for what a quantized
cache stores, bit for bit against kvf_b200_quantize of rows rotated in fp32
torch operations."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from kvforge_b200 import FMT_F16, FMT_INT4, FMT_INT8, ORD_HEAD, ORD_TOKEN, api  # noqa: E402
from kvforge_b200 import layout  # noqa: E402
from kvforge_b200.layout import Placement  # noqa: E402

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
EPS = 1e-6
PLACES = [Placement(ORD_HEAD, False, 0), Placement(ORD_TOKEN, False, 0), Placement(ORD_HEAD, True, 16),
          Placement(ORD_TOKEN, True, 32)]
FORMATS = [(FMT_F16, 0), (FMT_INT8, 64), (FMT_INT4, 32)]


def _gen(cuda, seed):
    g = torch.Generator(device=cuda)
    g.manual_seed(seed)
    return g


def _randn(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=g.device).to(dtype)


def _exact(x, pos, rope, weight):
    """The formulas in 64 bits: (y, sum of the magnitudes that each y adds)."""
    x = x.double()
    B, T, H, d = x.shape
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
    if rope is None:
        return x, x.abs()
    y, mag = x.clone(), x.abs()
    r = 2 * rope.cos.shape[1]
    a, b = (slice(0, r, 2), slice(1, r, 2)) if rope.interleaved else (slice(0, r // 2), slice(r // 2, r))
    for i in range(B):
        at = torch.arange(T, device=x.device) + int(pos[i])
        c, s = rope.cos[at].double()[:, None], rope.sin[at].double()[:, None]
        u, w = x[i, :, :, a], x[i, :, :, b]
        y[i, :, :, a], y[i, :, :, b] = u * c - w * s, u * s + w * c
        mag[i, :, :, a], mag[i, :, :, b] = (u * c).abs() + (w * s).abs(), (u * s).abs() + (w * c).abs()
    return y, mag


def _fp32(x, pos, rope, weight):
    """The same in fp32 torch operations, one rounding each, the squares in a tree of neighbours."""
    x = x.float()
    B, T, H, d = x.shape
    if weight is not None:
        s = x * x
        while s.shape[-1] > 1:
            s = s[..., 0::2] + s[..., 1::2]
        x = x * (1.0 / torch.sqrt(s / d + EPS)) * weight.float()
    if rope is None:
        return x
    y = x.clone()
    r = 2 * rope.cos.shape[1]
    at = pos[:, None].long() + torch.arange(T, device=x.device)
    c, s = rope.cos[at][:, :, None], rope.sin[at][:, :, None]
    a, b = (slice(0, r, 2), slice(1, r, 2)) if rope.interleaved else (slice(0, r // 2), slice(r // 2, r))
    u, w = x[..., a], x[..., b]
    y[..., a], y[..., b] = u * c - w * s, u * s + w * c
    return y


def _assert_formula(got, y, mag, dtype, what):
    """fp32 work: the mean of squares is off by at most 8 roundings (a square and
    7 sums), its root halves that to 4, root, sum with eps, reciprocal and the two
    products add 5, the rotation a product and a sum: 11 half steps of 2^-24 on
    each term added, taken as 12 for the second order. Then one rounding to the
    type: half of eps, relative; subnormals of fp16 by at most 2^-25."""
    err = (got.double() - y).abs()
    tol = 12 * 2.0 ** -24 * mag
    tol = tol + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2) * (y.abs() + tol) + 2.0 ** -25
    assert bool((err <= tol).all()), f"{what}: off by {float((err - tol).max()):.3g} more than the bound"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,rot,interleaved", [(128, 128, False), (128, 128, True), (128, 32, False), (128, 96, False),
                                               (128, 16, True), (64, 64, False), (64, 32, True), (64, 48, False)])
@pytest.mark.parametrize("norm", [False, True])
def test_norm_rope_matches_the_formula(cuda, dtype, d, rot, interleaved, norm):
    g = _gen(cuda, 1)
    B, T, H = 3, 7, 5
    rope = api.Rope.build(300, rot, interleaved=interleaved, device=cuda)
    weight = (1 + 0.2 * _randn((d,), g)).to(dtype) if norm else None
    pos = torch.tensor([0, 293, 40], dtype=torch.int32, device=cuda)
    x = _randn((B, T, H, d), g, dtype) * 3
    got = api.norm_rope(x, pos, rope, weight=weight, eps=EPS)
    assert api.device_errors() == 0 and got.dtype == dtype
    y, mag = _exact(x, pos, rope, weight)
    _assert_formula(got, y, mag, dtype, "norm_rope")
    assert torch.equal(got, _fp32(x, pos, rope, weight).to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_alone_and_long_batches(cuda, dtype):
    """Without rotation (no positions needed); enough rows for four per lane group."""
    g = _gen(cuda, 2)
    x = _randn((5, 301, 9, 128), g, dtype)
    w = _randn((128,), g)
    got = api.norm_rope(x, None, weight=w, eps=EPS)
    y, mag = _exact(x, None, None, w)
    _assert_formula(got, y, mag, dtype, "norm")
    x = _randn((2, 4000, 13, 64), g, dtype)
    rope = api.Rope.build(4100, 64, device=cuda)
    pos = torch.tensor([100, 3], dtype=torch.int32, device=cuda)
    assert torch.equal(api.norm_rope(x, pos, rope), _fp32(x, pos, rope, None).to(dtype))
    assert api.device_errors() == 0


def test_norm_rope_strides_lengths_and_in_place(cuda):
    g = _gen(cuda, 3)
    B, T, H, d = 4, 6, 3, 64
    rope = api.Rope.build(64, 64, device=cuda)
    pos = torch.tensor([5, 0, 50, 9], dtype=torch.int32, device=cuda)
    lens = torch.tensor([6, 0, 3, 100], dtype=torch.int32, device=cuda)  # 100 counts as T
    for off in (0, 1, 8):  # rows on and off 16-byte boundaries
        big = _randn((T, B, 2 * H * d + 9), g, torch.bfloat16)
        x = big[..., off: off + H * d].unflatten(-1, (H, d)).transpose(0, 1)
        want = _fp32(x, pos, rope, None).to(x.dtype)
        out = torch.full((B, T, H, d), 7.0, dtype=x.dtype, device=cuda)
        api.norm_rope(x, pos, rope, lens=lens, out=out)
        for b, m in enumerate((6, 0, 3, 6)):
            assert torch.equal(out[b, :m], want[b, :m])
            assert bool((out[b, m:] == 7.0).all())
        rest = big.clone()
        api.norm_rope(x, pos, rope, out=x)  # onto itself, through its strides
        assert torch.equal(x, want)
        rest[..., off: off + H * d] = big[..., off: off + H * d]
        assert torch.equal(rest, big)
    assert api.device_errors() == 0


def test_norm_rope_reports_positions_outside_the_table(cuda):
    g = _gen(cuda, 4)
    rope = api.Rope.build(10, 64, device=cuda)
    x = _randn((3, 2, 2, 64), g)
    pos = torch.tensor([9, -1, 2 ** 31 - 1], dtype=torch.int32, device=cuda)
    out = torch.full_like(x, 7.0)
    api.norm_rope(x, pos, rope, out=out)
    assert api.device_errors() == 4 and api.device_errors() == 0
    want = _fp32(x, torch.tensor([9, -1, 0], device=cuda).clamp(0, 8), rope, None)
    assert bool((out[0, 1] == 7.0).all()) and bool((out[1, 0] == 7.0).all()) and bool((out[2] == 7.0).all())
    assert torch.equal(out[1, 1], _fp32(x[1:2, 1:2], torch.tensor([0], device=cuda), rope, None)[0, 0])
    assert torch.equal(out[0, 0], _fp32(x[0:1, 0:1], torch.tensor([9], device=cuda), rope, None)[0, 0])
    assert want.shape == x.shape


def _empty_cache(cuda, B, Hkv, n, d, fmt, group, place, seed=5, seq_lens=None):
    z = torch.zeros((B, Hkv, n, d), device=cuda)
    return api.KVCache.from_logical(z, z, fmt=fmt, group=group, place=place, table_seed=seed, seq_lens=seq_lens)


def _expected(cache, before, k32, v32, pos, lens):
    """The buffers with the rows of k32, v32 [B][T][Hkv][D] quantized and placed by the host's row formula."""
    want = [None if t is None else t.clone() for t in before]
    table = cache.block_table.cpu().numpy() if cache.block_table is not None else None
    for which, x in ((0, k32), (1, v32)):
        data, meta = api.quantize(x.contiguous(), cache.fmt, cache.group)
        B, T, Hkv, d = x.shape
        rows, src = [], []
        for b in range(B):
            for j in range(lens[b]):
                t = pos[b] + j
                if t < 0 or t >= cache.n:
                    continue
                for h in range(Hkv):
                    rows.append(layout.row_of(cache.place.order, cache.place.block_tokens if cache.place.paged else 0,
                                              Hkv, cache.n, table, cache.max_blocks, b, h, t))
                    src.append((b * T + j) * Hkv + h)
        if rows:
            rows = torch.tensor(rows, device=x.device)
            src = torch.tensor(src, device=x.device)
            want[which][rows] = data[src]
            if meta is not None:
                want[2 + which][rows] = meta[src]
    return want


def _buffers(c):
    return [c.k, c.v, c.k_meta, c.v_meta]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("place", PLACES, ids=lambda p: p.name)
@pytest.mark.parametrize("fmt,group", FORMATS + [(FMT_INT8, 128), (FMT_INT4, 128)])
def test_append_rope_stores_the_quantized_rotated_rows(cuda, dtype, place, fmt, group):
    g = _gen(cuda, 6)
    B, T, H, Hkv, n, d = 3, 9, 10, 5, 70, 128
    cache = _empty_cache(cuda, B, Hkv, n, d, fmt, group, place)
    before = [None if t is None else t.clone() for t in _buffers(cache)]
    qkv = _randn((B, T, H + 2 * Hkv, d), g, dtype)
    q, k, v = qkv.split((H, Hkv, Hkv), 2)
    rope = api.Rope.build(n, 128, device=cuda)
    wk, wq = (1 + 0.1 * _randn((d,), g)).to(dtype), _randn((d,), g)
    pos, lens = [0, 61, 33], [9, 9, 4]
    dpos, dlens = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in (pos, lens))
    out = api.append_rope(cache, k, v, rope, pos=dpos, lens=dlens, k_weight=wk, q=q, q_weight=wq, eps=EPS)
    assert api.device_errors() == 0
    for got, want in zip(_buffers(cache), _expected(cache, before, _fp32(k, dpos, rope, wk), v.float(), pos, lens)):
        assert got is want is None or torch.equal(got, want)
    want = _fp32(q, dpos, rope, wq).to(dtype)
    for b, m in enumerate(lens):
        assert torch.equal(out[b, :m], want[b, :m]) and not out[b, m:].any()


@pytest.mark.parametrize("fmt,group", [(FMT_F16, 0), (FMT_INT8, 64), (FMT_INT4, 32), (FMT_INT4, 64)])
def test_append_rope_narrow_heads_partial_rotation(cuda, fmt, group):
    g = _gen(cuda, 7)
    B, T, Hkv, n, d = 2, 33, 3, 64, 64
    place = Placement(ORD_TOKEN, True, 16)
    cache = _empty_cache(cuda, B, Hkv, n, d, fmt, group, place)
    before = [None if t is None else t.clone() for t in _buffers(cache)]
    k, v = _randn((B, T, Hkv, d), g, torch.float16), _randn((B, T, Hkv, d), g, torch.float16)
    rope = api.Rope.build(n, 32, interleaved=True, device=cuda)
    pos = torch.tensor([31, 2], dtype=torch.int32, device=cuda)
    assert api.append_rope(cache, k, v, rope, pos=pos) is None
    for got, want in zip(_buffers(cache), _expected(cache, before, _fp32(k, pos, rope, None), v.float(), [31, 2], [33, 33])):
        assert got is want is None or torch.equal(got, want)
    assert api.device_errors() == 0


@pytest.mark.parametrize("fmt,group", FORMATS)
def test_append_rope_without_rotation_is_append(cuda, fmt, group):
    """Edge values too: constant groups, signed zeros, infinities, NaN, values past fp16."""
    g = _gen(cuda, 8)
    B, T, Hkv, n, d = 2, 6, 2, 40, 128
    k, v = _randn((B, T, Hkv, d), g), _randn((B, T, Hkv, d), g) * 1e-4
    k[0, 0] = 3.0
    k[0, 1, 0, :64] = 0.0
    k[0, 1, 0, 1:64:2] = -0.0
    k[0, 2, 0, 5] = float("inf")
    k[0, 2, 1, 70] = float("-inf")
    k[0, 3, 0, 0] = float("nan")
    k[0, 3, 1, 31] = float("nan")
    k[0, 4] *= 1e5
    k[0, 5] = 1e-9
    lens = np.array([11, 30], dtype=np.int32)
    place = Placement(ORD_TOKEN, False, 0)
    a = _empty_cache(cuda, B, Hkv, n, d, fmt, group, place, seq_lens=lens)
    c = _empty_cache(cuda, B, Hkv, n, d, fmt, group, place, seq_lens=lens)
    api.append(a, k.transpose(1, 2), v.transpose(1, 2))
    api.append_rope(c, k, v)
    for x, y in zip(_buffers(a), _buffers(c)):
        assert x is y is None or torch.equal(x, y)
    assert torch.equal(c.seq_lens, a.seq_lens)
    api.append_rope(c, k[:, :1], v[:, :1], lens=torch.tensor([1, 0], dtype=torch.int32, device=cuda))
    assert c.seq_lens.tolist() == [18, 36]
    assert api.device_errors() == 0


def test_append_rope_skips_what_has_no_row(cuda):
    g = _gen(cuda, 9)
    B, T, Hkv, n, d = 3, 4, 2, 32, 64
    cache = _empty_cache(cuda, B, Hkv, n, d, FMT_INT8, 64, Placement(ORD_HEAD, True, 16))
    cache.block_table[2, 0] = -1
    before = [t.clone() for t in _buffers(cache)]
    k, v = _randn((B, T, Hkv, d), g), _randn((B, T, Hkv, d), g)
    pos = torch.tensor([30, -2, 14], dtype=torch.int32, device=cuda)
    api.append_rope(cache, k, v, pos=pos)
    assert api.device_errors() == 4 and api.device_errors() == 0
    # written: tokens 30, 31 of sequence 0; 0, 1 of sequence 1; 16, 17 of sequence 2 (14, 15 have no page)
    k2, v2 = k.clone(), v.clone()
    want = _expected(cache, before, k2[:2], v2[:2], [30, -2], [4, 4])
    want = _expected(cache, want, torch.cat((k2[:2] * 0, k2[2:, 2:].expand(1, 2, Hkv, d).repeat(1, 2, 1, 1))),
                     torch.cat((v2[:2] * 0, v2[2:, 2:].expand(1, 2, Hkv, d).repeat(1, 2, 1, 1))), [0, 0, 16], [0, 0, 2])
    for got, w in zip(_buffers(cache), want):
        assert torch.equal(got, w)
    short = api.Rope.build(17, 64, device=cuda)  # a table that ends inside the chunk
    api.append_rope(cache, k, v, short, pos=torch.tensor([0, 0, 16], dtype=torch.int32, device=cuda), lens=None)
    assert api.device_errors() == 4


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("place", PLACES, ids=lambda p: p.name)
@pytest.mark.parametrize("fmt,group,d", [(FMT_F16, 0, 128), (FMT_INT8, 64, 128), (FMT_INT8, 128, 128),
                                         (FMT_INT4, 32, 128), (FMT_INT4, 64, 64), (FMT_F16, 0, 64)])
def test_gather_reads_what_is_stored(cuda, dtype, place, fmt, group, d):
    """Against zero + scale * code in 64 bits: the product has at most 19 bits, so
    fp32 rounds once; a 16-bit type once more."""
    g = _gen(cuda, 10)
    B, Hkv, n, T = 3, 5, 70, 21
    K, V = _randn((B, Hkv, n, d), g), _randn((B, Hkv, n, d), g) * 5
    cache = api.KVCache.from_logical(K, V, fmt=fmt, group=group, place=place)
    pos, lens = [0, 49, 13], [21, 21, 5]
    out = [torch.full((B, T, Hkv, d), 7.0, dtype=dtype, device=cuda) for _ in range(2)]
    api.gather(cache, T, pos=torch.tensor(pos, dtype=torch.int32, device=cuda),
               lens=torch.tensor(lens, dtype=torch.int32, device=cuda), out=out)
    assert api.device_errors() == 0
    for X, got in zip((K, V), out):
        data, meta = api.quantize(X, fmt, group)
        if fmt == FMT_F16:
            y = data.view(torch.float16).double()
        else:
            c = data.double() if fmt == FMT_INT8 else torch.stack((data & 15, data >> 4), -1).flatten(-2).double()
            sz = meta.view(torch.float16).double().unflatten(-1, (-1, 2))
            y = c * sz[..., 0].repeat_interleave(group, -1) + sz[..., 1].repeat_interleave(group, -1)
        y = y.reshape(B, Hkv, n, d).transpose(1, 2)
        for b in range(B):
            want, have = y[b, pos[b]: pos[b] + lens[b]], got[b, : lens[b]].double()
            rel = 2.0 ** -24 + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -20))
            assert bool(((have - want).abs() <= rel * want.abs() + 2.0 ** -25).all())
            assert bool((got[b, lens[b]:] == 7.0).all())


def test_gather_stops_at_lengths_and_reports_tokens_without_a_row(cuda):
    g = _gen(cuda, 11)
    B, Hkv, n, d = 3, 2, 48, 64
    K = _randn((B, Hkv, n, d), g)
    lens = np.array([48, 20, 0], dtype=np.int32)
    cache = api.KVCache.from_logical(K, K, fmt=FMT_F16, place=Placement(ORD_TOKEN, True, 16), seq_lens=lens)
    k, v = api.gather(cache, n)
    for b, m in enumerate(lens):
        assert torch.equal(k[b, :m], K[b, :, :m].transpose(0, 1).half().float()) and not k[b, m:].any()
    assert torch.equal(k, v) and api.device_errors() == 0
    api.gather(cache, 4, pos=torch.tensor([46, 0, 0], dtype=torch.int32, device=cuda))  # ends with the sequence
    assert api.device_errors() == 0
    cache.seq_lens = None
    api.gather(cache, 4, pos=torch.tensor([46, 0, -1], dtype=torch.int32, device=cuda))  # past n, before 0
    assert api.device_errors() == 4
    odd = torch.zeros((B, 5, Hkv, d + 1), dtype=torch.bfloat16, device=cuda)
    out = (odd[..., 1:], torch.zeros((B, 5, Hkv, d), dtype=torch.bfloat16, device=cuda))
    cache.seq_lens = torch.tensor([48, 20, 0], dtype=torch.int32, device=cuda)
    api.gather(cache, 5, out=out)  # rows off 16-byte boundaries
    assert torch.equal(out[0], out[1]) and not odd[..., 0].any()
    assert torch.equal(out[1][0], K[0, :, :5].transpose(0, 1).half().to(torch.bfloat16))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,H,interleaved", [(128, 64, False), (128, 61, True), (64, 64, False), (64, 20, False), (128, 3, False)])
def test_long_calls_match_short_ones(cuda, dtype, d, H, interleaved):
    """Enough tokens for several rows per lane, against calls of few tokens and the fp32 operations."""
    g = _gen(cuda, 14)
    B, T = 2, 1300
    rope = api.Rope.build(T + 10, d, interleaved=interleaved, device=cuda)
    w = 1 + 0.1 * _randn((d,), g)
    pos = torch.tensor([7, 0], dtype=torch.int32, device=cuda)
    x = _randn((B, T, H, d), g, dtype)
    got = api.norm_rope(x, pos, rope, weight=w, eps=EPS)
    assert torch.equal(got, _fp32(x, pos, rope, w).to(dtype))
    at = pos + 1000
    assert torch.equal(got[:, 1000:1003], api.norm_rope(x[:, 1000:1003], at, rope, weight=w, eps=EPS))
    odd = torch.zeros((B, T, H * d + 1), dtype=dtype, device=cuda)[..., 1:].unflatten(-1, (H, d))
    assert torch.equal(got, api.norm_rope(x, pos, rope, weight=w, eps=EPS, out=odd))  # rows off 16-byte boundaries
    assert api.device_errors() == 0


@pytest.mark.parametrize("fmt,group,d", [(FMT_F16, 0, 128), (FMT_INT8, 64, 128), (FMT_INT4, 32, 128), (FMT_INT4, 32, 64)])
@pytest.mark.parametrize("Hkv", [1, 2, 8, 11])
def test_long_append_and_gather(cuda, fmt, group, d, Hkv):
    g = _gen(cuda, 15)
    B, T, n = 2, 1200, 1300
    place = Placement(ORD_TOKEN, True, 16)
    cache = _empty_cache(cuda, B, Hkv, n, d, fmt, group, place)
    k, v = (_randn((B, T, Hkv, d), g, torch.bfloat16) for _ in range(2))
    q = _randn((B, T, 4 * Hkv, d), g, torch.bfloat16)
    rope = api.Rope.build(n, d, device=cuda)
    pos = torch.tensor([100, 3], dtype=torch.int32, device=cuda)
    out = api.append_rope(cache, k, v, rope, pos=pos, q=q)
    assert torch.equal(out, _fp32(q, pos, rope, None).to(q.dtype))
    got = api.gather(cache, T, pos=pos)
    for x, y in zip((_fp32(k, pos, rope, None), v.float()), got):
        data, meta = api.quantize(x.contiguous(), fmt, group)
        one = api.KVCache(fmt=fmt, d=d, group=group, place=Placement(ORD_TOKEN, False, 0), B=B, Hkv=Hkv, n=T, k=data, v=data,
                          k_meta=meta, v_meta=meta, block_table=None, max_blocks=0, seq_lens=None)
        assert torch.equal(y, api.gather(one, T)[0])
    assert api.device_errors() == 0


def test_offsets_past_32_bits(cuda):
    """Pages far into a pool of more than 4 GB: payload and metadata offsets need 64 bits."""
    g = _gen(cuda, 16)
    B, T, Hkv, n, d, pages = 1, 20, 2, 32, 128, 1_100_000
    for fmt, group in ((FMT_INT8, 64), (FMT_F16, 0)):
        pages = 1_100_000 if fmt == FMT_INT8 else 600_000
        rows = pages * Hkv * 16
        k, v = (torch.zeros((rows, api.row_bytes(fmt, d)), dtype=torch.uint8, device=cuda) for _ in range(2))
        assert k.numel() > 2 ** 32
        km, vm = (torch.zeros((rows, 2), dtype=torch.int32, device=cuda) if group else None for _ in range(2))
        table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device=cuda)
        cache = api.KVCache(fmt=fmt, d=d, group=group, place=Placement(ORD_TOKEN, True, 16), B=B, Hkv=Hkv, n=n, k=k, v=v,
                            k_meta=km, v_meta=vm, block_table=table, max_blocks=2,
                            seq_lens=torch.tensor([T], dtype=torch.int32, device=cuda))
        kn, vn = (_randn((B, T, Hkv, d), g, torch.bfloat16) for _ in range(2))
        api.append_rope(cache, kn, vn, pos=torch.zeros(B, dtype=torch.int32, device=cuda))
        small = _empty_cache(cuda, B, Hkv, n, d, fmt, group, Placement(ORD_TOKEN, False, 0),
                             seq_lens=np.array([T], dtype=np.int32))
        api.append_rope(small, kn, vn, pos=torch.zeros(B, dtype=torch.int32, device=cuda))
        for x, y in zip(api.gather(cache, T), api.gather(small, T)):
            assert torch.equal(x, y) and bool(x.any())
        for dtype in (torch.bfloat16, torch.float32):
            q = _randn((B, T, 8, d), g, dtype)
            assert torch.equal(api.chunk_attention(q, cache), api.chunk_attention(q, small))
        assert api.device_errors() == 0
        del k, v, km, vm, cache


def test_heads_on_another_stream_and_in_a_graph(cuda):
    g = _gen(cuda, 12)
    B, T, H, Hkv, n, d = 2, 3, 4, 2, 32, 128
    cache = _empty_cache(cuda, B, Hkv, n, d, FMT_INT8, 64, Placement(ORD_TOKEN, True, 16))
    cache.seq_lens = torch.zeros(B, dtype=torch.int32, device=cuda)  # every page mapped, no token stored yet
    rope = api.Rope.build(n, 128, device=cuda)
    qkv = _randn((B, T, H + 2 * Hkv, d), g, torch.bfloat16)
    q, k, v = qkv.split((H, Hkv, Hkv), 2)
    q_out, vals = torch.zeros_like(q), [torch.zeros((B, T, Hkv, d), device=cuda) for _ in range(2)]
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    x = api.norm_rope(q, cache.seq_lens, rope, stream=side)
    side.synchronize()
    zero = torch.zeros(B, dtype=torch.int32, device=cuda)
    assert torch.equal(x, _fp32(q, zero, rope, None).to(q.dtype))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        api.append_rope(cache, k, v, rope, q=q, q_out=q_out)
        api.gather(cache, T, out=vals)
    assert cache.seq_lens.tolist() == [0, 0]
    for step in range(3):
        qkv.copy_(_randn(qkv.shape, g, qkv.dtype))
        graph.replay()
        at = torch.full((B,), step * T, dtype=torch.int32, device=cuda)
        assert cache.seq_lens.tolist() == [T * (step + 1)] * B
        assert torch.equal(q_out, _fp32(q, at, rope, None).to(q.dtype))
        if step == 0:
            first = _fp32(k, at, rope, None)
        assert float((vals[0] - first).abs().max()) < 0.05  # a code's half step of groups spanning about 6
    assert api.device_errors() == 0


def test_refusals(cuda):
    g = _gen(cuda, 13)
    rope = api.Rope.build(16, 64, device=cuda)
    x = _randn((2, 3, 2, 64), g)
    pos = torch.zeros(2, dtype=torch.int32, device=cuda)
    cache = _empty_cache(cuda, 2, 2, 16, 64, FMT_INT8, 64, Placement(ORD_TOKEN, False, 0))
    bad = [
        lambda: api.norm_rope(x, pos),
        lambda: api.norm_rope(x, None, rope),
        lambda: api.norm_rope(x[0], pos, rope),
        lambda: api.norm_rope(x.double(), pos, rope),
        lambda: api.norm_rope(x.transpose(2, 3), pos, rope),
        lambda: api.norm_rope(x, pos.long(), rope),
        lambda: api.norm_rope(x, pos[:1], rope),
        lambda: api.norm_rope(x, pos.cpu(), rope),
        lambda: api.norm_rope(x, pos, rope, out=x.half()),
        lambda: api.norm_rope(x, pos, rope, weight=x[0, 0, 0, :32]),
        lambda: api.Rope(rope.cos.double(), rope.sin.double()),
        lambda: api.Rope(rope.cos, rope.sin[:, :8]),
        lambda: api.Rope(rope.cos.t(), rope.sin.t()),
        lambda: api.append_rope(cache, x[:, :, :1], x, pos=pos),
        lambda: api.append_rope(cache, x, x.half(), pos=pos),
        lambda: api.append_rope(cache, x, x),
        lambda: api.append_rope(cache, x, x, pos=pos, q_weight=x[0, 0, 0]),
        lambda: api.append_rope(cache, x, x, pos=pos, q=x[:, :2]),
        lambda: api.gather(cache, 4, out=(x, x.half())),
        lambda: api.gather(cache, 4, out=(x, x)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"case {i} was taken")
    short = api.Rope(torch.zeros((16, 4), device=cuda), torch.zeros((16, 4), device=cuda))  # rot = 8
    with pytest.raises(api.KvfError):
        api.norm_rope(x, pos, short)
    with pytest.raises(api.KvfError):
        api.norm_rope(x[..., :32], pos, rope)  # 32 channels
    assert api.norm_rope(x[:0], pos[:0], rope).numel() == 0
    assert api.norm_rope(x[:, :0], pos, rope).numel() == 0
    assert api.device_errors() == 0
