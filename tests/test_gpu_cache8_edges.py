"""Decode attention over the 8-bit cache where V's exponents are far apart, and what the calls of the
8-bit cache share: plans, streams, workspaces."""
from __future__ import annotations

import numpy as np
import pytest

from cache8_model import D
from test_gpu_cache8 import DEV, cache8, dev, rows  # noqa: F401 (fixture)
from test_gpu_window_edges import cached, far_pages, weighed

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("step,zero", [(12, 1), (24, 1), (40, 1), (70, 1), (-24, 1), (-70, 1), (24, 0), (-40, 0),
                                       (105, 0), (115, 1)])
@pytest.mark.parametrize("G,lens", [(8, [150]), (1, [33]), (8, [1100]), (2, [4000]), (8, [5, 16, 47, 300, 111]),
                                    (8, [200] * 20 + [700])])
def test_decode_goes_by_the_v_that_weighs(cache8, step, zero, G, lens):
    """V pages 2^step apart in turn, with pages of zeros among them where `zero` is 0; the pages of large V
    weigh 2^-(step + 16) in every second slot, and must then not cost the others their bits."""
    rng = np.random.default_rng(101)
    c = cache8(G=G, n_pages=1200, max_slots=32)
    slots = []
    # the heads of a slot are close to one direction, along which the pages of large V lie backwards
    q = np.repeat(rng.standard_normal((len(lens), 1, D)), 4 * G, 1) + 0.1 * rng.standard_normal((len(lens), 4 * G, D))
    q = q.astype(np.float32)
    for i, n in enumerate(lens):
        s = c.slot(n + 1)
        k, v = rows(rng, n, G), far_pages(rng, n, G, step, zero)
        if i % 2 == 0 and step > 0:
            turned = c.rope(q[i:i + 1], [n])[0, ::4]
            back = -(step + 16) * np.log(2) * np.sqrt(float(D)) / (turned ** 2).sum(-1, keepdims=True) * turned
            for p in range(1, (n + 15) // 16, 2):
                k[16 * p:16 * p + 16] = 0.05 * k[16 * p:16 * p + 16] + back
        c.eng.qkv_write(0, [s], [n], None, dev(k), dev(v), rotated=True)
        c.eng.advance([s], n)
        slots.append(s)
    n = len(slots)
    k, v = rows(rng, n, G), rows(rng, n, G)
    out, again = torch.empty((2, n, 4 * G * D), device=DEV).unbind(0)
    c.eng.decode_step(0, slots, dev(q), dev(k), dev(v), out)
    c.eng.decode_attn(0, slots, dev(q), again)
    c.eng.sync_check()
    assert torch.equal(out, again)
    out = out.double().cpu().numpy().reshape(n, 4 * G, D)
    for i in range(0, n, 4):
        p = lens[i]
        kk, vv = cached(c.eng, c.hkv, slots[i], p + 1, G)
        x = c.rope(q[i:i + 1], [p]).astype(np.float64)
        want, bound = weighed(x, kk, vv, p, "f32", 14)
        over = np.abs(out[i:i + 1] - want) - bound
        assert over.max() <= 0, (i, np.unravel_index(over.argmax(), over.shape), over.max())


@pytest.mark.parametrize("lens", [[900], [3, 200, 31], [100] * 20])
def test_decode_of_values_near_the_largest_floats(cache8, lens):
    """V of up to 3e38 everywhere: a mean, not infinity, in every way partials are merged."""
    rng = np.random.default_rng(103)
    c = cache8(G=8, n_pages=1200, max_slots=32)
    slots = []
    for n in lens:
        s = c.slot(n + 1)
        v = (rng.uniform(1.0, 3.0, (n, 8, D)) * 1e38).astype(np.float32)
        c.eng.rope_append_range(0, s, n, dev(rows(rng, n, 8)), dev(v))
        c.eng.advance([s], n)
        slots.append(s)
    n = len(slots)
    q = rng.standard_normal((n, 32, D)).astype(np.float32)
    v = (rng.uniform(1.0, 3.0, (n, 8, D)) * 1e38).astype(np.float32)
    out = torch.empty((n, 32 * D), device=DEV)
    c.eng.decode_step(0, slots, dev(q), dev(rows(rng, n, 8)), dev(v), out)
    out = out.double().cpu().numpy().reshape(n, 32, D)
    for i in range(0, n, 7):
        kk, vv = cached(c.eng, c.hkv, slots[i], lens[i] + 1, 8)
        want, bound = weighed(c.rope(q[i:i + 1], [lens[i]]).astype(np.float64), kk, vv, lens[i], "f32", 14)
        assert (np.abs(out[i:i + 1] - want) <= bound).all(), i


def test_a_failed_call_does_not_fail_the_next(cache8):
    """A call that needs an allocation while a stream captures is refused by CUDA; the error is that call's
    alone."""
    rng = np.random.default_rng(107)
    c = cache8(G=1)
    s = c.slot()
    c.prefill(s, rows(rng, 20, 1), rows(rng, 20, 1))
    k, v = torch.zeros((2, 20, 1, D), dtype=torch.int16, device=DEV).unbind(0)
    side, work = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    failed = False
    with torch.cuda.stream(side):
        graph.capture_begin()
        try:
            c.eng.gather(s, 0, 0, 20, k, v, stream=work.cuda_stream)
        except c.hkv.HkvError as e:
            failed = e.status == c.hkv.HKV_ERR_CUDA
        try:
            graph.capture_end()
        except RuntimeError:
            pass  # the refused allocation ended the capture
    if failed:
        c.eng.gather(s, 0, 0, 20, k, v, stream=work.cuda_stream)
    work.synchronize()
    want, _ = c.read(s, 0, 20, dtype=torch.float16)
    assert np.array_equal(k.cpu().numpy().view(np.float16), want)


@pytest.mark.parametrize("low,high", [(0.0, 1e12), (0.0, 1e30), (1e-25, 1e20), (1e25, 0.0)])
@pytest.mark.parametrize("G,lens", [(8, [700]), (1, [700]), (8, [650, 640, 300]), (8, [640] * 20), (8, [1900] * 30), (1, [31000])])
def test_decode_where_v_jumps(cache8, low, high, G, lens):
    """The first 256 rows' V far below, or above, that of the others, at like weights."""
    rng = np.random.default_rng(123)
    c = cache8(G=G, n_pages=4000, max_slots=32)
    slots = []
    for n in lens:
        s = c.slot(n + 1)
        v = rows(rng, n, G)
        v[:256] *= np.float32(low)
        v[256:] *= np.float32(high)
        c.eng.rope_append_range(0, s, n, dev(rows(rng, n, G) * np.float32(0.3)), dev(v))
        c.eng.advance([s], n)
        slots.append(s)
    n = len(slots)
    q = rng.standard_normal((n, 4 * G, D)).astype(np.float32)
    out = torch.empty((n, 4 * G * D), device=DEV)
    c.eng.decode_step(0, slots, dev(q), dev(rows(rng, n, G)), dev(rows(rng, n, G) * np.float32(high)), out)
    out = out.double().cpu().numpy().reshape(n, 4 * G, D)
    for i in range(0, n, 6):
        kk, vv = cached(c.eng, c.hkv, slots[i], lens[i] + 1, G)
        want, bound = weighed(c.rope(q[i:i + 1], [lens[i]]).astype(np.float64), kk, vv, lens[i], "f32", 14)
        over = np.abs(out[i:i + 1] - want) - bound
        assert over.max() <= 0, (i, np.unravel_index(over.argmax(), over.shape), over.max())
