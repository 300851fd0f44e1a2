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
@pytest.mark.parametrize("rows", [2, 70])
def test_infinite_keys_and_values(cuda, dtype, rows):
    """A key whose score is -inf has weight 0 and no other effect; a value that is
    infinite makes its column infinite for the rows that see it; a key whose
    score is +inf makes the row NaN. In whole steps and in masked ones."""
    g = _gen(cuda, 3)
    B, T, H, Hkv, n, d = 1, rows, 4, 2, 700, 128
    K, V = _randn((B, Hkv, n, d), g), _randn((B, Hkv, n, d), g)
    q = _randn((B, T, H, d), g).abs().add(0.01)
    q[..., 1] *= -1
    q = q.to(dtype)
    gone = [3, 300, n - T - 1, n - T + 1 if T > 2 else n - T]
    want_v = V.clone()
    for t in gone:
        K[..., t, 0] = -math.inf
        K[..., t, 1] = math.inf if t == 300 else 1.0  # negative queries: also -inf
    cols = {17: (200, math.inf), 18: (n - T, -math.inf), 19: (n - 1, math.inf), 64: (0, -math.inf)}
    for c, (t, x) in cols.items():
        want_v[..., t, c] = 0
        V[..., t, c] = x
    for place in (HEAD, TOKEN16):
        cache = api.KVCache.from_logical(K, V, fmt=FMT_F16, place=place)
        k, v = (x.double() for x in api.gather(cache, n))
        plain = v.clone().nan_to_num(0.0, 0.0, 0.0)
        for splits in (1, 2, 3):
            got = _attend(q, cache, splits)
            for h in range(H):
                s = (q[0, :, h].double() @ k[0, :, h // 2].T).div(math.sqrt(d))
                last = n - T + torch.arange(T, device=cuda)
                hidden = torch.arange(n, device=cuda) > last[:, None]
                p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
                assert not p.isnan().any() and not p[:, gone].any()
                want = p @ plain[0, :, h // 2]
                for c, (t, x) in cols.items():
                    want[last >= t, c] = x if t not in gone else math.nan
                fine, inf = want.isfinite(), want.isinf()
                mine = got[0, :, h].double()
                assert torch.equal(mine.isfinite(), fine), f"splits {splits}"
                tol = 2.0 ** -14 if dtype == torch.float32 else 2.0 ** -7
                assert bool(((mine - want)[fine].abs() <= tol).all())
                if dtype == torch.float32:  # 16-bit queries: infinite or NaN, since their weights are rounded (0 * inf)
                    assert torch.equal(mine[inf], want[inf]) and torch.equal(mine.isnan(), want.isnan())
    K[..., 400, 0] = math.inf
    cache = api.KVCache.from_logical(K, V, fmt=FMT_F16, place=TOKEN16)
    for splits in (1, 2):
        assert bool(_attend(q, cache, splits).isnan().all())
    assert api.device_errors() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt,group,d", [(FMT_INT8, 64, 128), (FMT_INT4, 32, 128), (FMT_INT8, 64, 64), (FMT_INT4, 64, 64)])
@pytest.mark.parametrize("rows", [3, 70])
def test_quantized_values_past_fp16(cuda, dtype, fmt, group, d, rows):
    """Groups of a quantized cache that hold values past 65504, or whose scale or
    zero is infinite, at late tokens: rows that do not see them are those of a
    cache without them, bit for bit or in another order of the same sums."""
    g = _gen(cuda, 4)
    B, T, H, Hkv, n = 2, rows, 4, 2, 500
    K, V = _randn((B, Hkv, n, d), g), _randn((B, Hkv, n, d), g)
    lens = [500, 389]
    K2, V2 = K.clone(), V.clone()
    first = []
    for b, kv in enumerate(lens):
        K2[b, :, kv:], V2[b, :, kv:] = 1e30, -1e30            # nobody's
        V2[b, 0, kv - 1, : group] = torch.linspace(0, 2e5, group, device=cuda)   # finite, past fp16
        V2[b, 1, kv - 1, : group] = torch.linspace(-1e30, 1e30, group, device=cuda)  # scale and zero infinite
        K2[b, 1, kv - 1, d - group:] = torch.linspace(-1e30, 1e30, group, device=cuda)
        first.append(kv - 1)
    for place in (HEAD, TOKEN16):
        a = api.KVCache.from_logical(K, V, fmt=fmt, group=group, place=place)
        c = api.KVCache.from_logical(K2, V2, fmt=fmt, group=group, place=place)
        a.seq_lens = c.seq_lens = torch.tensor(lens, dtype=torch.int32, device=cuda)
        q = _randn((B, T, H, d), g, dtype)
        for splits in (1, 2, 3, 4):
            x, y = _attend(q, a, splits), _attend(q, c, splits)
            tol = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -9 if dtype == torch.float16 else 2.0 ** -17
            early, late = slice(0, T - 1), T - 1
            assert bool(y[:, early].isfinite().all()), f"splits {splits}"
            assert bool(((x - y)[:, early].abs() <= tol * (x[:, early].abs() + 1)).all()), f"splits {splits}"
            # the last row of heads 0, 1 sees values up to 2e5, heads 2, 3 a NaN key
            assert bool(y[:, late, 2:].isnan().all())
            big = y[:, late, :2, : group]
            assert bool(y[:, late, :2, group:].isfinite().all())
            if dtype == torch.float32:
                assert bool(big.isfinite().all()) and bool((big[..., -1] > 0).all())
            else:
                assert bool((big[..., -1] == math.inf).all()) and bool(big[..., 0].isfinite().all())
    assert api.device_errors() == 0


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


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("fmt,group", [(FMT_F16, 0), (FMT_INT8, 64)])
def test_the_greatest_query(cuda, dtype, fmt, group):
    """A channel of the type's greatest number against zero keys adds nothing."""
    g = _gen(cuda, 8)
    B, T, H, Hkv, n, d = 1, 9, 4, 2, 200, 64
    K = _randn((B, Hkv, n, d), g).abs()  # a group's least value is its zero point: zero is stored as zero
    K[..., 5] = 0
    cache = api.KVCache.from_logical(K, _randn((B, Hkv, n, d), g), fmt=fmt, group=group, place=TOKEN)
    q = _randn((B, T, H, d), g, dtype)
    q[..., 5] = 0
    want = api.chunk_attention(q, cache)
    q[..., 5] = torch.finfo(dtype).max
    assert torch.equal(api.chunk_attention(q, cache), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("splits", [1, 2, 3])
def test_nan_queries(cuda, dtype, splits):
    """A NaN query's row is NaN, and so is its lse (-inf is for rows that see nothing)."""
    g = _gen(cuda, 5)
    B, T, H, Hkv, n, d = 2, 5, 4, 2, 300, 64
    cache = api.KVCache.from_logical(_randn((B, Hkv, n, d), g), _randn((B, Hkv, n, d), g), fmt=FMT_INT8, group=64, place=TOKEN16)
    cache.seq_lens = torch.tensor([300, 3], dtype=torch.int32, device=cuda)
    q = _randn((B, T, H, d), g, dtype)
    clean_lse = torch.zeros((B, T, H), device=cuda)
    clean = _attend(q, cache, splits, lse=clean_lse)
    bad = torch.zeros((B, T, H), dtype=torch.bool, device=cuda)
    bad[0, 1, 2] = bad[1, 4, 0] = bad[1, 0, 1] = True  # the last one sees nothing
    q[bad] = math.nan
    lse = torch.zeros((B, T, H), device=cuda)
    got = _attend(q, cache, splits, lse=lse)
    sees = clean_lse > -math.inf
    assert bool(got[bad & sees].isnan().all()) and bool(lse[bad & sees].isnan().all())
    assert not got[bad & ~sees].any() and bool((lse[bad & ~sees] == -math.inf).all())
    assert torch.equal(got[~bad], clean[~bad]) and torch.equal(lse[~bad], clean_lse[~bad])


@pytest.mark.parametrize("fmt,group,d", [(FMT_INT8, 64, 128), (FMT_INT4, 32, 128)])
def test_metadata_on_odd_words(cuda, fmt, group, d):
    """fp32 queries read metadata by words: any 4-byte address will do. 16-bit
    queries need a row's words on their own alignment."""
    g = _gen(cuda, 6)
    B, T, H, Hkv, n = 1, 3, 2, 1, 50
    cache = api.KVCache.from_logical(_randn((B, Hkv, n, d), g), _randn((B, Hkv, n, d), g), fmt=fmt, group=group, place=TOKEN)
    q = _randn((B, T, H, d), g)
    want = api.chunk_attention(q, cache)
    for name in ("k_meta", "v_meta"):
        m = getattr(cache, name)
        odd = torch.zeros(m.numel() + 1, dtype=m.dtype, device=cuda)[1:].view(m.shape)
        odd.copy_(m)
        setattr(cache, name, odd)
    assert torch.equal(api.chunk_attention(q, cache), want)
    with pytest.raises(api.KvfError):
        api.chunk_attention(q.half(), cache)


def test_workspace_for_what_is_stored(cuda):
    """A long cache that holds little: splits by the lengths that are to come, and
    right for longer ones."""
    g = _gen(cuda, 9)
    B, T, H, Hkv, n, d = 1, 16, 8, 2, 20000, 128
    cache = api.KVCache.from_logical(_randn((B, Hkv, n, d), g), _randn((B, Hkv, n, d), g), fmt=FMT_F16, place=TOKEN)
    q = _randn((B, T, H, d), g, torch.bfloat16)
    assert api.ChunkWorkspace.allocate(cache, T, H, q.dtype).splits > 4
    ws = api.ChunkWorkspace.allocate(cache, T, H, q.dtype, n=100)
    assert ws.splits == 1 and ws.part_o is None
    for length in (100, n):
        cache.seq_lens = torch.tensor([length], dtype=torch.int32, device=cuda)
        a, b = api.chunk_attention(q, cache, workspace=ws), api.chunk_attention(q, cache)
        # weights and their sums are rounded alike, but summed in another order: a step of bf16 apart at most
        assert bool(((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 2.0 ** -10).all())


def test_workspaces_that_do_not_hold_the_partials(cuda):
    """Of another type, with gaps, or too small: refused, since the kernels write all of it."""
    g = _gen(cuda, 10)
    B, T, H, Hkv, n, d = 1, 8, 4, 2, 500, 64
    cache = api.KVCache.from_logical(_randn((B, Hkv, n, d), g), _randn((B, Hkv, n, d), g), fmt=FMT_F16, place=TOKEN)
    q = _randn((B, T, H, d), g, torch.bfloat16)
    good = api.ChunkWorkspace.allocate(cache, T, H, q.dtype, splits=4)
    wide = torch.zeros((*good.part_o.shape[:-1], 2 * d), device=cuda)
    for part_o, part_ml in ((good.part_o.half(), good.part_ml), (good.part_o, good.part_ml.half()), (wide[..., ::2], good.part_ml),
                            (good.part_o[:, :-1], good.part_ml), (good.part_o.cpu(), good.part_ml)):
        with pytest.raises(ValueError):
            api.chunk_attention(q, cache, workspace=api.ChunkWorkspace(4, part_o, part_ml))
    assert bool(api.chunk_attention(q, cache, workspace=good).isfinite().all()) and api.device_errors() == 0


def _softmax_rows(q, cache):
    """Causal attention over the stored values in 64 bits, whole sequences of n tokens."""
    B, T, H, d = q.shape
    k, v = (x.double() for x in api.gather(cache, cache.n))
    g, n = H // cache.Hkv, cache.n
    k, v = (x.repeat_interleave(g, 2).transpose(1, 2) for x in (k, v))
    s = q.double().transpose(1, 2) @ k.transpose(-1, -2) / math.sqrt(d)
    last = n - T + torch.arange(T, device=q.device)
    s.masked_fill_(torch.arange(n, device=q.device) > last[:, None], -math.inf)
    return (torch.softmax(s, -1) @ v).transpose(1, 2)


def _near(got, want):
    """Normal inputs of 128 channels or fewer. 16-bit queries: keys off by 2^-11 move a
    score by at most 2^-11 sum |q k| / sqrt(d), about 2^-11 * 8, and the output by twice
    that times its |values| (about 1): 2^-7; weights, values and the output's rounding add
    2^-9 at most. fp32: 2^-21 in place of 2^-11, and sums over the tokens."""
    tol = 2.0 ** -14 if got.dtype == torch.float32 else 2.0 ** -6
    return bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt,group", [(FMT_F16, 0), (FMT_INT8, 64), (FMT_INT4, 32)])
@pytest.mark.parametrize("order", [ORD_HEAD, ORD_TOKEN])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_every_page_size(cuda, dtype, fmt, group, order, page):
    g = _gen(cuda, 11)
    B, T, H, Hkv, n, d = 2, 40, 6, 3, 300, 128
    cache = api.KVCache.from_logical(_randn((B, Hkv, n, d), g), _randn((B, Hkv, n, d), g), fmt=fmt, group=group,
                                     place=Placement(order, True, page))
    q = _randn((B, T, H, d), g, dtype)
    want = _softmax_rows(q, cache)
    for splits in (1, 2, 3):
        assert _near(_attend(q, cache, splits), want)
    assert api.device_errors() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [100, 129, 300, 5000])
def test_many_query_heads_for_a_kv_head(cuda, dtype, heads):
    """Tiles that end inside a token's heads, and tokens of many tiles."""
    g = _gen(cuda, 12)
    B, T, Hkv, n, d = 1, 3, 2, 150, 64
    cache = api.KVCache.from_logical(_randn((B, Hkv, n, d), g), _randn((B, Hkv, n, d), g), fmt=FMT_INT8, group=64, place=TOKEN16)
    q = _randn((B, T, heads * Hkv, d), g, dtype)
    want = _softmax_rows(q, cache)
    for splits in (1, 2):
        assert _near(_attend(q, cache, splits), want)
    assert api.device_errors() == 0


def test_calls_on_two_streams_at_once(cuda):
    """Chunks of two batches on streams of their own, default workspaces: the bits of calls one by one."""
    g = _gen(cuda, 13)
    B, T, H, Hkv, n, d = 4, 16, 16, 4, 3000, 128
    sets = []
    for fmt, group, dtype in ((FMT_INT8, 64, torch.bfloat16), (FMT_F16, 0, torch.float32)):
        cache = api.KVCache.from_logical(_randn((B, Hkv, n, d), g), _randn((B, Hkv, n, d), g), fmt=fmt, group=group, place=TOKEN16)
        q = _randn((B, T, H, d), g, dtype)
        assert api.ChunkWorkspace.allocate(cache, T, H, dtype).splits > 1
        sets.append((q, cache, api.chunk_attention(q, cache), torch.cuda.Stream(cuda)))
    torch.cuda.synchronize()
    for _ in range(20):
        outs = [api.chunk_attention(q, cache, stream=st) for q, cache, _, st in sets]
        torch.cuda.synchronize()
        for x, (_, _, want, _) in zip(outs, sets):
            assert torch.equal(x, want)
    assert api.device_errors() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt,group,d", [(FMT_F16, 0, 128), (FMT_F16, 0, 64), (FMT_INT8, 64, 128), (FMT_INT4, 32, 64)])
@pytest.mark.parametrize("page", [16, 64, 128])
def test_seen_blocks_without_a_page_are_zeros(cuda, dtype, fmt, group, d, page):
    """In the middle and at the end of a sequence, whatever earlier steps left behind."""
    g = _gen(cuda, 14)
    B, T, H, Hkv, n = 2, 30, 4, 2, 500
    cache = api.KVCache.from_logical(_randn((B, Hkv, n, d), g), _randn((B, Hkv, n, d), g), fmt=fmt, group=group,
                                     place=Placement(ORD_HEAD, True, page))
    cache.block_table[0, 1] = cache.block_table[1, 0] = cache.block_table[1, -1] = -1
    q = _randn((B, T, H, d), g, dtype)
    want = _softmax_rows(q, cache)  # reads such blocks back as zeros, and reports them
    assert api.device_errors() == 4
    for splits in (1, 2, 3):
        assert _near(_attend(q, cache, splits), want)
    assert api.device_errors() == 0


def test_a_stream_of_small_calls(cuda):
    """Many short calls of all kinds, one behind the other: sequences of no, one and
    few tokens, splits without tokens, pages that end inside a tile."""
    import random

    g, rng = _gen(cuda, 15), random.Random(15)
    results = []
    for _ in range(150):
        d, fmt = rng.choice((64, 128)), rng.choice((FMT_F16, FMT_INT8, FMT_INT4))
        B, T, Hkv, heads, n = rng.choice((1, 2, 5)), rng.randint(1, 40), rng.choice((1, 2, 3)), rng.choice((1, 2, 5)), rng.randint(1, 200)
        page = rng.choice((0, 16, 64, 128))
        cache = api.KVCache.empty(B, Hkv, n, d, fmt=fmt, group=0 if fmt == FMT_F16 else 64,
                                  place=Placement(rng.choice((ORD_HEAD, ORD_TOKEN)), page > 0, page), device=cuda)
        k, v = (_randn((B, n, Hkv, d), g, torch.float16) for _ in range(2))
        kv = torch.randint(0, n + 1, (B,), generator=g, device=cuda, dtype=torch.int32)
        api.append_rope(cache, k, v, lens=kv)
        q = _randn((B, T, heads * Hkv, d), g, rng.choice(DTYPES))
        lens = torch.randint(0, T + 1, (B,), generator=g, device=cuda, dtype=torch.int32)
        outs = [_attend(q, cache, s, q_lens=lens) for s in (1, 2, 4, 7)]
        results.append((outs, d))
    for outs, d in results:
        for x in outs[1:]:
            # rows of one token or a few: values up to about 5, rounded alike or one step of the type apart
            tol = 1e-4 if x.dtype == torch.float32 else 2.0 ** -8 if x.dtype == torch.float16 else 2.0 ** -5
            assert bool(x.isfinite().all()) and bool(((x.float() - outs[0].float()).abs() <= tol).all())
    assert api.device_errors() == 0
