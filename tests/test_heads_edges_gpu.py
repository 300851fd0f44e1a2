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


def _rotated(x, pos, rope, weight):
    """norm_rope in fp32 torch operations, one rounding each, the squares in a tree of neighbours."""
    x = x.float()
    T, d = x.shape[1], x.shape[-1]
    if weight is not None:
        s = x * x
        while s.shape[-1] > 1:
            s = s[..., 0::2] + s[..., 1::2]
        x = x * (1.0 / torch.sqrt(s / d + 1e-6)) * weight.float()
    if rope is None:
        return x
    y, r = x.clone(), 2 * rope.cos.shape[1]
    at = pos[:, None].long() + torch.arange(T, device=x.device)
    c, s = rope.cos[at][:, :, None], rope.sin[at][:, :, None]
    u, w = x[..., : r // 2], x[..., r // 2: r]
    y[..., : r // 2], y[..., r // 2: r] = u * c - w * s, u * s + w * c
    return y


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,heads,d,rot", [
    (2100, 8, 128, 128), (2100, 8, 128, 64), (5000, 16, 128, 128), (5000, 16, 128, 64), (5000, 15, 128, 128),
    (2100, 16, 64, 64), (5000, 32, 64, 64), (5000, 32, 64, 32), (5000, 31, 64, 64), (1, 3, 128, 128)])
def test_every_number_of_rows_per_lane(cuda, dtype, T, heads, d, rot):
    """Long calls take two, four (fp32) or eight (16-bit) rows per lane group, by how
    many heads fill them; rotated whole or in part, normed or not."""
    g = _gen(cuda, 1)
    B = 3
    x = _randn((B, T, heads, d), g, dtype)
    w = (1 + 0.1 * _randn((d,), g)).to(dtype)
    rope = api.Rope.build(T + 50, rot, device=cuda)
    pos = torch.tensor([0, 49, 7], dtype=torch.int32, device=cuda)
    for weight, r in ((None, rope), (w, rope), (w, None)):
        got = api.norm_rope(x, None if r is None else pos, r, weight=weight)
        assert torch.equal(got, _rotated(x, pos, r, weight).to(dtype))
    assert api.device_errors() == 0


def test_rows_beside_a_position_outside_the_table(cuda):
    """What is inside is rotated as ever, in every row."""
    g = _gen(cuda, 2)
    rope = api.Rope.build(10, 64, device=cuda)
    x = _randn((3, 4, 2, 64), g)
    pos = torch.tensor([8, -2, 3], dtype=torch.int32, device=cuda)
    out = torch.full_like(x, 7.0)
    api.norm_rope(x, pos, rope, out=out)
    assert api.device_errors() == 4 and api.device_errors() == 0
    for b in range(3):
        for t in range(4):
            p = int(pos[b]) + t
            want = torch.full_like(x[b, t], 7.0)
            if 0 <= p < 10:
                want = _rotated(x[b: b + 1, t: t + 1], torch.tensor([p], device=cuda), rope, None)[0, 0]
            assert torch.equal(out[b, t], want)

@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("order", [ORD_HEAD, ORD_TOKEN])
def test_append_past_the_mapped_blocks(cuda, fmt, group, order):
    """A cache built with lengths maps the blocks of stored tokens only: tokens
    appended past those are skipped and reported, and no other sequence's page is
    touched."""
    g = _gen(cuda, 3)
    B, Hkv, n, d = 3, 2, 80, 64
    lens = [33, 1, 16]
    K, V = _randn((B, Hkv, n, d), g), _randn((B, Hkv, n, d), g)
    group = min(group, d)
    for call in ("append", "append_rope"):
        cache = api.KVCache.from_logical(K, V, fmt=fmt, group=group, place=Placement(order, True, 16), seq_lens=lens)
        before = api.gather(cache, n)
        T = 20
        k, v = _randn((B, T, Hkv, d), g), _randn((B, T, Hkv, d), g)
        if call == "append":
            api.append(cache, k.transpose(1, 2), v.transpose(1, 2))
        else:
            api.append_rope(cache, k, v)
        assert api.device_errors() == 4
        # the mapped blocks hold 48, 16 and 16 tokens: 15, 15 and 0 of the 20 fit
        cache.seq_lens = torch.tensor([48, 16, 16], dtype=torch.int32, device=cuda)
        after = api.gather(cache, n)
        assert api.device_errors() == 0
        kq, vq = (api.KVCache.from_logical(x.transpose(1, 2).contiguous(), x.transpose(1, 2).contiguous(), fmt=fmt, group=group,
                                           place=Placement(ORD_TOKEN, False, 0)) for x in (k, v))
        for was, now, new in zip(before, after, (api.gather(kq, T)[0], api.gather(vq, T)[0])):
            for b, (m, fit) in enumerate(zip(lens, (15, 15, 0))):
                assert torch.equal(now[b, :m], was[b, :m])
                assert torch.equal(now[b, m: m + fit], new[b, :fit])


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


@pytest.mark.parametrize("fmt,group", FORMATS)
@pytest.mark.parametrize("place", [Placement(ORD_HEAD, False, 0), Placement(ORD_TOKEN, True, 16)], ids=lambda p: p.name)
def test_an_empty_cache_is_filled(cuda, fmt, group, place):
    """KVCache.empty holds no tokens and room for n of every sequence: filled by
    append_rope it is the cache that from_logical makes."""
    g = _gen(cuda, 5)
    B, H, Hkv, n, d = 3, 8, 2, 50, 128
    cache = api.KVCache.empty(B, Hkv, n, d, fmt=fmt, group=group, place=place, device=cuda)
    assert cache.seq_lens.tolist() == [0] * B and cache.payload_bytes() == 0
    q = _randn((B, H, d), g)
    assert not api.decode(q, cache).any()
    k, v = _randn((B, n, Hkv, d), g), _randn((B, n, Hkv, d), g)
    lens = torch.tensor([17, 0, 50], dtype=torch.int32, device=cuda)
    api.append_rope(cache, k, v, lens=lens)
    assert cache.seq_lens.tolist() == [17, 0, 50]
    rest = [(17, 33), (0, 50), (50, 0)]
    pad = torch.zeros_like(k), torch.zeros_like(v)
    for b, (m, r) in enumerate(rest):
        for x, y in zip(pad, (k, v)):
            x[b, :r] = y[b, m:]
    api.append_rope(cache, *pad, lens=torch.tensor([r for _, r in rest], dtype=torch.int32, device=cuda))
    assert cache.seq_lens.tolist() == [n] * B and api.device_errors() == 0
    full = api.KVCache.from_logical(k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous(), fmt=fmt, group=group,
                                    place=place)
    for x, y in zip(api.gather(cache, n), api.gather(full, n)):
        assert torch.equal(x, y)
    assert float((api.decode(q, cache) - api.decode(q, full)).abs().max()) < 1e-5


def test_tensors_that_want_gradients_are_refused(cuda):
    """No call around the cache has a backward pass: a graph would end here without a word."""
    g = _gen(cuda, 6)
    B, T, H, Hkv, n, d = 1, 3, 4, 2, 16, 64
    cache = api.KVCache.empty(B, Hkv, n, d, fmt=FMT_F16, place=Placement(ORD_TOKEN, False, 0), device=cuda)
    q, k, v = _randn((B, T, H, d), g), _randn((B, T, Hkv, d), g), _randn((B, T, Hkv, d), g)
    w = torch.ones(d, device=cuda)
    pos = torch.zeros(B, dtype=torch.int32, device=cuda)

    def wants(x):
        return x.clone().requires_grad_()

    calls = [lambda f: api.norm_rope(f(q), None, weight=w), lambda f: api.norm_rope(q, None, weight=f(w)),
             lambda f: api.norm_rope(q, None, weight=w, out=f(q)),
             lambda f: api.append_rope(cache, f(k), v, pos=pos), lambda f: api.append_rope(cache, k, f(v), pos=pos),
             lambda f: api.append_rope(cache, k, v, pos=pos, k_weight=f(w)),
             lambda f: api.append_rope(cache, k, v, pos=pos, q=f(q), q_weight=w),
             lambda f: api.append_rope(cache, k, v, pos=pos, q=q, q_weight=f(w)),
             lambda f: api.append_rope(cache, k, v, pos=pos, q=q, q_out=f(q)),
             lambda f: api.gather(cache, T, out=(f(k), v)),
             lambda f: api.chunk_attention(f(q), cache), lambda f: api.chunk_attention(q, cache, out=f(q))]
    for call in calls:
        with pytest.raises(ValueError, match="backward"):
            call(wants)
        call(lambda x: x)
        with torch.no_grad():
            call(wants)
    assert api.device_errors() == 0


def test_a_step_in_a_graph(cuda):
    """append_rope that raises the lengths itself, and attention with a workspace of the
    graph's own, replayed: the bits of calls one by one."""
    g = _gen(cuda, 7)
    B, T, H, Hkv, n, d = 3, 2, 8, 2, 64, 128
    place = Placement(ORD_TOKEN, True, 16)
    a, b = (api.KVCache.empty(B, Hkv, n, d, fmt=FMT_INT8, group=64, place=place, device=cuda) for _ in range(2))
    rope = api.Rope.build(n, d, device=cuda)
    qkv = _randn((B, T, H + 2 * Hkv, d), g, torch.bfloat16)
    q, k, v = qkv.split((H, Hkv, Hkv), 2)
    lens = torch.tensor([2, 1, 2], dtype=torch.int32, device=cuda)

    def step(cache):
        return api.chunk_attention(api.append_rope(cache, k, v, rope, q=q, lens=lens), cache, q_lens=lens)

    step(a)  # kernels' attributes are set outside the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a)
    a.seq_lens.zero_()
    for x in (a.k, a.v, a.k_meta, a.v_meta):
        x.zero_()
    for new in ([2, 1, 2], [1, 0, 2], [2, 2, 2], [0, 1, 1]):
        qkv.copy_(_randn(qkv.shape, g, qkv.dtype))
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, step(b))
        assert torch.equal(a.seq_lens, b.seq_lens)
    for x, y in zip((a.k, a.v, a.k_meta, a.v_meta), (b.k, b.v, b.k_meta, b.v_meta)):
        assert torch.equal(x, y)
    assert api.device_errors() == 0
