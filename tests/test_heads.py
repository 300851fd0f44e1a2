"""kvf_b200_norm_rope, kvf_b200_append_rope and kvf_b200_gather refuse what they
cannot do before anything touches a GPU."""
from __future__ import annotations

import ctypes

import pytest

from kvforge_b200._native import KvfArgs, KvfHeads, KvfNorm, KvfRope, lib

FAKE = 0x1000  # never dereferenced: every case fails or returns before a launch
INVALID, MISALIGNED = 1, 716


def heads(**kw):
    return KvfHeads(**{**dict(p=FAKE, dtype=2, heads=8, stride_b=1024, stride_t=1024, stride_h=128), **kw})


def rope(**kw):
    return KvfRope(**{**dict(cos=FAKE, sin=FAKE, positions=64, rot=128, interleaved=0), **kw})


def cache(**kw):
    a = KvfArgs()
    a.k = a.v = a.k_meta = a.v_meta = a.block_table = FAKE
    a.B, a.H, a.Hkv, a.n, a.group_shift, a.block_shift, a.max_blocks = 2, 8, 8, 64, 6, 4, 4
    for name, v in kw.items():
        setattr(a, name, v)
    return a


def ref(x):
    return None if x is None else ctypes.byref(x)


def norm_rope(x=None, out=None, B=2, T=3, d=128, r="rope", norm=None, pos=FAKE):
    r = rope() if r == "rope" else r
    return lib().kvf_b200_norm_rope(ref(x or heads()), ref(out or heads()), B, T, d, ref(r), ref(norm), pos, None, None)


def test_norm_rope_checks():
    assert norm_rope(T=0) == 0 and norm_rope(B=0) == 0
    for kw in (dict(B=-1), dict(T=-1), dict(d=96), dict(r=None), dict(pos=None), dict(x=heads(dtype=3)),
               dict(x=heads(dtype=-1)), dict(x=heads(p=None)), dict(x=heads(heads=0)), dict(out=heads(dtype=1)),
               dict(out=heads(heads=4)), dict(r=rope(rot=120)), dict(r=rope(rot=144)), dict(r=rope(rot=0)),
               dict(r=rope(positions=0)), dict(r=rope(interleaved=2)), dict(r=rope(cos=None)),
               dict(norm=KvfNorm(None, 0, 1e-6)), dict(norm=KvfNorm(FAKE, 5, 1e-6)), dict(norm=KvfNorm(FAKE, 0, -1.0)),
               dict(norm=KvfNorm(FAKE, 0, float("nan")))):
        assert norm_rope(**kw) == INVALID, kw
    for kw in (dict(x=heads(p=FAKE + 1)), dict(r=rope(sin=FAKE + 4)), dict(norm=KvfNorm(FAKE + 2, 0, 1e-6))):
        assert norm_rope(**kw) == MISALIGNED, kw


def append(a=None, fmt=1, d=128, ord=1, paged=1, k=None, v=None, T=3, pos=FAKE, q=None, qo=None, qn=None):
    a = cache() if a is None else a
    return lib().kvf_b200_append_rope(ref(a), fmt, d, ord, paged, ref(k or heads()), ref(v or heads()), T, None, None,
                                      pos, None, ref(q), ref(qo), ref(qn), None)


def gather(a=None, fmt=1, d=128, ord=1, paged=1, T=3, k=None, v=None):
    a = cache() if a is None else a
    return lib().kvf_b200_gather(ref(a), fmt, d, ord, paged, T, None, None, ref(k or heads()), ref(v or heads()), None)


@pytest.mark.parametrize("call", [append, gather])
def test_cache_checks(call):
    assert call(T=0) == 0 and call(a=cache(B=0)) == 0
    for kw in (dict(T=-1), dict(fmt=3), dict(fmt=-1), dict(d=96), dict(ord=2), dict(paged=2), dict(a=cache(B=-1)),
               dict(a=cache(Hkv=0)), dict(a=cache(n=0)), dict(a=cache(group_shift=4)), dict(a=cache(group_shift=5)),
               dict(a=cache(group_shift=8)), dict(a=cache(group_shift=7), d=64), dict(a=cache(k=None)),
               dict(a=cache(v_meta=None)), dict(a=cache(block_table=None)), dict(a=cache(max_blocks=0)),
               dict(a=cache(block_shift=-1)), dict(k=heads(heads=4)), dict(v=heads(dtype=0)), dict(v=heads(p=None))):
        assert call(**kw) == INVALID, kw
    for kw in (dict(a=cache(k=FAKE + 8)), dict(a=cache(k_meta=FAKE + 2)), dict(v=heads(p=FAKE + 1))):
        assert call(**kw) == MISALIGNED, kw
    assert lib().kvf_b200_gather(None, 1, 128, 1, 1, 3, None, None, ref(heads()), ref(heads()), None) == INVALID


def test_append_query_checks():
    q = heads(heads=32)
    for kw in (dict(pos=None), dict(q=q), dict(qo=q), dict(q=q, qo=heads(heads=16)), dict(q=heads(dtype=0), qo=heads(dtype=0)),
               dict(q=q, qo=heads(heads=32, dtype=0)), dict(qn=KvfNorm(FAKE, 0, 1e-6))):
        assert append(**kw) == INVALID, kw


def chunk(a=None, fmt=1, d=128, ord=1, paged=1, q=None, out=None, T=3, causal=1):
    a = cache(H=32, splits=1) if a is None else a
    q = q or heads(heads=32)
    return lib().kvf_b200_chunk_attention(ref(a), fmt, d, ord, paged, ref(q), ref(out or heads(heads=32)), T, None, causal,
                                          None)


def test_chunk_attention_checks():
    good = dict(H=32, splits=1)
    assert chunk(T=0) == 0 and chunk(a=cache(B=0, **good)) == 0
    for kw in (dict(T=-1), dict(causal=2), dict(causal=-1), dict(fmt=3), dict(d=96), dict(ord=2), dict(paged=2),
               dict(a=cache(H=30, splits=1)), dict(a=cache(H=32, splits=0)), dict(a=cache(H=0, splits=1)),
               dict(a=cache(H=32, splits=2)), dict(a=cache(max_blocks=3, **good)), dict(a=cache(k=None, **good)),
               dict(a=cache(group_shift=5, **good)), dict(q=heads(heads=16)), dict(out=heads(heads=32, dtype=1)),
               dict(out=heads(heads=16)), dict(q=heads(heads=32, p=None)), dict(T=1 << 30),
               dict(a=cache(n=(1 << 30) + 1, max_blocks=1 << 27, **good)), dict(q=heads(heads=32, stride_t=1 << 30)),
               dict(out=heads(heads=32, stride_h=1 << 30)), dict(a=cache(block_shift=3, **good)),
               dict(a=cache(block_shift=8, **good)), dict(a=cache(H=8 * 65536, splits=1), q=heads(heads=8 * 65536),
                                                          out=heads(heads=8 * 65536))):
        assert chunk(**kw) == INVALID, kw
    for kw in (dict(a=cache(v=FAKE + 4, **good)), dict(out=heads(heads=32, p=FAKE + 1)),
               dict(a=cache(H=32, splits=2, part_o=FAKE + 4, part_ml=FAKE))):
        assert chunk(**kw) == MISALIGNED, kw


def test_chunk_splits_needs_no_gpu():
    f = lib().kvf_b200_chunk_splits
    assert f(0, 1, 8, 8, 100, 0, 128, 0) == 1 and f(1, 1, 8, 3, 100, 0, 128, 0) == 1
    assert f(1, 1, 8, 8, 100, 0, 128, 2) >= 1 and f(1, 4, 32, 8, 65536, 1, 128, 2) > 8
    assert f(64, 4096, 32, 8, 65536, 1, 128, 2) == 1
