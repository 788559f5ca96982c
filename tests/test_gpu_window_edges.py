"""hkv_window_attn on the GPU where it can go wrong: rows whose scales differ, rows and pages of
zeros, pages of V far apart, workspaces and plans that calls share.

Held to float64 over the rows that the cache holds, as test_gpu_window.py does.
"""
from __future__ import annotations

import numpy as np
import pytest

from cache8_model import D
from test_gpu_cache8 import DEV, dev, rows
from test_gpu_window import DT, check, engine, fill, window

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", ["e4m3", "f16"])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_rows_of_different_scales(hkv_lib, cache, name):
    """Rows of q from 2^-9 to 2^2, another power for each row and head, in both halves of every tile:
    each row keeps its own scale, and thirty launches give the same bits."""
    import hkv
    rng = np.random.default_rng(83)
    G = 8
    eng = engine(hkv, G, cache)
    s = eng.acquire()
    fill(eng, rng, s, 19, G)
    fill(eng, rng, s, 200, G, advance=False)
    scale = np.exp2(rng.integers(-9, 3, (200, 4 * G, 1)))
    q = torch.from_numpy((rng.standard_normal((200, 4 * G, D)) * scale).astype(np.float32)).to(DEV)
    out = window(eng, hkv, [s], [200], q, name)
    check(eng, hkv, [s], [200], q, out, name)
    again = torch.empty_like(out)
    x = q.to(DT[name])
    for _ in range(30):
        eng.window_attn(0, [s], [200], x, again, dtype=getattr(hkv, name.upper()))
        assert torch.equal(out, again)
    eng.close()
