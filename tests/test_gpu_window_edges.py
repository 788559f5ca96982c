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


@pytest.mark.parametrize("cache", ["e4m3", "f16"])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_zero_rows_give_the_mean(hkv_lib, cache, name):
    """Zero q, zero K, both, and both close to nothing: every logit is 0, so a row is the mean of the V it
    sees.  Slots that end inside a page and a block, behind a prefix and without one."""
    import hkv
    rng = np.random.default_rng(85)
    G = 2
    eng = engine(hkv, G, cache)
    old, new = [0, 770, 0, 13], [37, 70, 130, 1]
    tiny = 1e-30 if name != "f16" else 6e-8
    for zero_k, zero_q in ((1, 1), (1, 0), (0, 1), (1e-30, tiny)):
        slots = [eng.acquire() for _ in old]
        for s, p, n in zip(slots, old, new):
            for m, go_on in ((p, True), (n, False)):
                if m:
                    k = rows(rng, m, G) * np.float32(1 if not zero_k else 0 if zero_k == 1 else zero_k)
                    eng.rope_append_range(0, s, m, dev(k), dev(rows(rng, m, G)))
                    if go_on:
                        eng.advance([s], m)
        q = rng.standard_normal((sum(new), 4 * G, D)) * (1 if not zero_q else 0 if zero_q == 1 else zero_q)
        q = torch.from_numpy(q.astype(np.float32)).to(DEV)
        out = window(eng, hkv, slots, new, q, name)
        assert torch.isfinite(out).all(), (zero_k, zero_q)
        check(eng, hkv, slots, new, q, out, name)
        for s in slots:
            eng.release(s)
    eng.close()


def test_zero_rows_among_others(hkv_lib):
    """BF16 on an 8-bit cache: rows of zeros, as padding leaves them, in a batch of others; K pages of
    zeros in front of, in and behind the diagonal."""
    import hkv
    rng = np.random.default_rng(87)
    G, n = 1, 150
    eng = engine(hkv, G, "e4m3")
    s = eng.acquire()
    k, v = rows(rng, n, G), rows(rng, n, G)
    k[16:32] = k[64:80] = k[128:144] = 0
    v[32:48] = 0
    eng.rope_append_range(0, s, n, dev(k), dev(v))
    q = rng.standard_normal((n, 4 * G, D)).astype(np.float32)
    q[::3] = 0
    q = torch.from_numpy(q).to(DEV)
    check(eng, hkv, [s], [n], q, window(eng, hkv, [s], [n], q, "bf16"), "bf16")
    eng.close()
