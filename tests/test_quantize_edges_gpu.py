"""The device quantizer against the host's (oracle/kvf_oracle.c, kvf::quantize at
runtime/kvf_host.h:72-120) where its rules are easy to miss: signed zeros in
either order, NaN at the start of a group and inside it, infinities, constant
groups, values on the border between two codes, ranges past fp16."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import oracle as O

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from kvforge_b200 import FMT_INT4, FMT_INT8, api  # noqa: E402


def _rows(d, group, levels, rs):
    X = rs.standard_normal((400, d)).astype(np.float32)
    X[0] = 0.0
    X[1] = -0.0
    X[2, ::2], X[2, 1::2] = 0.0, -0.0
    X[3, ::2], X[3, 1::2] = -0.0, 0.0
    X[4] = np.abs(X[4])
    X[4, 5::7], X[4, 3::7] = 0.0, -0.0           # the least value is a zero of either sign
    X[5] = np.abs(X[5])
    X[5, 3::7], X[5, 6::7] = -0.0, 0.0
    X[6] = -np.abs(X[6])
    X[6, 1::5], X[6, 2::5] = 0.0, -0.0           # the greatest value is
    X[7, ::group] = np.nan                       # NaN first
    X[8, 3::group] = np.nan                      # NaN inside
    X[9] = np.nan
    X[10, group // 2::group] = np.inf
    X[11, group - 1::group] = -np.inf
    X[12, ::group], X[12, 1::group] = np.inf, -np.inf
    X[13] = 3.25
    X[14] = -7e4                                  # past fp16
    X[15] *= 1e5
    X[16] *= 1e30
    X[17] = 1e-9
    X[18] *= 1e-6                                 # subnormal fp16 scales
    X[19] *= 1e-42                                # subnormal fp32 values
    X[20, 1::2] = X[20, 0::2]
    # every half-integer border: a group from 0 to `levels` has scale 1 and zero 0
    for k in range(21, 200):
        X[k] = (rs.randint(0, 2 * levels + 1, size=d) / 2).astype(np.float32)
        X[k, ::group], X[k, 1::group] = 0.0, float(levels)
    for k in range(200, 300):                     # and just beside
        X[k] = np.nextafter((rs.randint(0, 2 * levels + 1, size=d) / 2).astype(np.float32),
                            np.float32(rs.choice([-1e9, 1e9])))
        X[k, ::group], X[k, 1::group] = -1.0, float(levels - 1)
    return X


@pytest.mark.parametrize("fmt,levels", [(FMT_INT8, 255), (FMT_INT4, 15)])
@pytest.mark.parametrize("d,group", [(128, 128), (128, 64), (128, 32), (128, 16), (128, 8), (64, 64), (64, 32), (64, 8)])
def test_edges_match_the_host(cuda, fmt, levels, d, group):
    X = _rows(d, group, levels, np.random.RandomState(41))
    want, meta, _ = O.quantize(fmt, d, group, X)
    got, gmeta = api.quantize(torch.as_tensor(X, device=cuda), fmt, group)
    assert np.array_equal(got.cpu().numpy(), want)
    # a NaN's payload is not part of the format
    a, b = gmeta.cpu().numpy().view(np.float16), meta.view(np.float16).reshape(gmeta.shape[0], -1)
    assert np.array_equal(np.isnan(a), np.isnan(b))
    assert np.array_equal(a.view(np.uint16)[~np.isnan(a)], b.view(np.uint16)[~np.isnan(b)])
