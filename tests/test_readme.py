"""The example under "Use" of the project's front page runs as it stands."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

PAGE = Path(__file__).resolve().parent.parent / "README.md"


def test_the_example_runs(cuda):
    text = re.search(r"## Use\n+```python\n(.*?)```", PAGE.read_text(), re.S).group(1)
    g = torch.Generator(device=cuda)
    g.manual_seed(1)
    B, H, Hkv, n, d, T = 2, 8, 2, 100, 128, 7

    def randn(*shape):
        return torch.randn(shape, generator=g, device=cuda)

    names = dict(K=randn(B, Hkv, n, d), V=randn(B, Hkv, n, d), q=randn(B, H, d), q_host=randn(B, H, d).cpu(), H=H, B=B,
                 Hkv=Hkv, n=n, k=randn(B, T, Hkv, d), v=randn(B, T, Hkv, d), q_new=randn(B, T, H, d))
    exec(compile(text, "example", "exec"), names)
    torch.cuda.synchronize()
    from kvforge_b200 import api

    assert names["out"].shape == (B, T, H, d) and bool(names["out"].isfinite().all()) and api.device_errors() == 0
