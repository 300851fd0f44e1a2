"""Groups whose least value is zero, whole warps of them, against the host's
quantizer (oracle/kvf_oracle.c): rows of zeros, of values from zero up, with the
one negative zero that decides a zero point's sign in any place of a group."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import oracle as O

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from kvforge_b200 import FMT_INT4, FMT_INT8, api  # noqa: E402


@pytest.mark.parametrize("fmt", [FMT_INT8, FMT_INT4])
@pytest.mark.parametrize("d,group", [(128, 64), (128, 32), (64, 64), (64, 8)])
@pytest.mark.parametrize("which", ["positive", "zeros", "negative zeros", "one negative zero", "nan"])
def test_zero_minima(cuda, fmt, d, group, which):
    rs = np.random.RandomState(7)
    X = np.maximum(rs.standard_normal((333, d)), 0).astype(np.float32) + np.float32(0)
    if which != "positive":
        X[:] = 0
    if which == "negative zeros":
        X[:] = -0.0
    for r in range(X.shape[0]):
        c = r % group
        if which == "one negative zero":
            X[r, c::group] = -0.0
            X[r, (c + 3) % d] = 1.0
        if which == "nan":
            X[r, c::group] = np.nan
            X[r, (c + 5) % d] = 2.0
    want, meta, _ = O.quantize(fmt, d, group, X)
    got, gmeta = api.quantize(torch.as_tensor(X, device=cuda), fmt, group)
    assert np.array_equal(got.cpu().numpy(), want)
    a, b = gmeta.cpu().numpy().view(np.float16), meta.view(np.float16).reshape(gmeta.shape[0], -1)
    assert np.array_equal(np.isnan(a), np.isnan(b))
    assert np.array_equal(a.view(np.uint16)[~np.isnan(a)], b.view(np.uint16)[~np.isnan(b)])
