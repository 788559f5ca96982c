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


def cached(eng, hkv, slot, n, G, layer=0):
    """Rows [0, n) of a slot as float64."""
    k, v = torch.empty((2, n, G, D), device=DEV).unbind(0)
    eng.cache_read(layer, [slot], [0], [n], k, v, dtype=hkv.F32)
    torch.cuda.synchronize()
    return k.double().cpu().numpy(), v.double().cpu().numpy()


def weighed(q, k, v, first, dtype, spare):
    """Float64 attention of rows q [T][H][D] over the rows k, v [L][G][D] and, for each output, a bound that
    goes by what the row weighs, not by the largest V of the slot.

    A weight is off relative to itself as attention_tolerance() derives (big: the largest sum_d |q_d k_d| * scale
    of the row), so an output by twice that times sum_t p_t |V_t| of its dim; F32 sums add 2^-23 of that for
    each 16 rows.  F16 and BF16 tensors round weights to F16: 2^-11 more.  Weights are held in F16 in
    units in which the largest p_t 2^eV of the row is at least 2^spare, to 2^-25 (half the least F16): each key
    adds up to 2^-(25 + spare) max_t(p_t 448 2^eV), and 448 * 2^eV is under twice the largest |V| of its page."""
    T, H, _ = q.shape
    L, G, _ = k.shape
    page = np.zeros((L, G))
    for p in range(0, L, 16):
        page[p:p + 16] = 2 * np.abs(v[p:p + 16]).max((0, 2))
    out, bound = np.zeros((T, H, D)), np.zeros((T, H, D))
    for h in range(H):
        g = h // (H // G)
        for i in range(T):
            n = first + i + 1
            s = k[:n, g] @ q[i, h] / np.sqrt(float(D))
            big = float((np.abs(k[:n, g]) @ np.abs(q[i, h])).max()) / np.sqrt(float(D))
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h] = p @ v[:n, g]
            rel = 2 * (big * (2.0 ** -22 + 2.0 ** -19) + 2 * big * 2.0 ** -23 + 2.0 ** -21 + 2.0 ** -22)
            if dtype != "f32":
                rel += 2 * 2.0 ** -11
            if dtype == "bf16":  # q in two E4M3 parts: 2^-10 / 224 of the row's largest a dim
                rel += 2 * np.abs(q[i, h]).max() * 2.0 ** -10 / 224 * np.abs(k[:n, g]).sum(-1).max() / np.sqrt(float(D))
            size = p @ np.abs(v[:n, g])
            bound[i, h] = size * (rel + (n / 16 + 64) * 2.0 ** -23) + n * 2.0 ** -(25 + spare) * (p * page[:n, g]).max()
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[dtype]
    return out, bound + half * (np.abs(out) + bound) + (2.0 ** -25 if dtype == "f16" else 0.0)


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


def test_logits_near_the_largest_floats(hkv_lib):
    """BF16 on an 8-bit cache: K of 1e37 against q of 0.01, logits of up to 1e35, each row one key's V; a
    product of codes and one exponent alone would overflow."""
    import hkv
    rng = np.random.default_rng(89)
    G, n = 1, 100
    eng = engine(hkv, G, "e4m3")
    s = eng.acquire()
    eng.rope_append_range(0, s, n, dev(rows(rng, n, G) * 1e36), dev(rows(rng, n, G)))
    q = torch.from_numpy((rng.standard_normal((n, 4 * G, D)) * 0.01).astype(np.float32)).to(DEV)
    out = window(eng, hkv, [s], [n], q, "bf16").double().cpu().numpy().reshape(n, 4, D)
    k, v = cached(eng, hkv, s, n, G)
    x = q.bfloat16().double().cpu().numpy()
    sure = 0
    for i in range(n):
        for h in range(4):
            a = np.sort(k[:i + 1, 0] @ x[i, h])[::-1]
            # q is held to 2^-17 of its largest value in each dim
            slack = 2.0 ** -17 * np.abs(x[i, h]).max() * np.abs(k[:i + 1, 0]).sum(-1).max() * 2
            if len(a) == 1 or a[0] - a[1] > 4 * slack:
                want = v[np.argmax(k[:i + 1, 0] @ x[i, h]), 0]
                assert (np.abs(out[i, h] - want) <= 2.0 ** -8 * np.abs(want)).all(), (i, h)
                sure += 1
    assert sure > 300
    eng.close()


STEPS = [(12, 1), (24, 1), (40, 1), (70, 1), (-24, 1), (-70, 1), (24, 0), (-40, 0), (105, 0)]


def far_pages(rng, n, G, step, zero):
    """V pages whose sizes alternate 2^step apart, with pages of zeros between them where `zero` is 0."""
    v = rows(rng, n, G).astype(np.float64)
    for p in range((n + 15) // 16):
        v[16 * p:16 * p + 16] *= 2.0 ** (step if p % 2 else 0) if zero or p % 3 else 0.0
    return v.astype(np.float32)


@pytest.mark.parametrize("step,zero", STEPS)
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_window_goes_by_the_v_it_sees(hkv_lib, name, step, zero):
    """V pages far apart in one tile: a row before a page of large V does not know of it, and a page that
    weighs nothing takes no bits from one that does.  Split (one slot) and whole tiles (16 slots of 8 heads)."""
    import hkv
    if name == "f16" and step > 12:
        step = 12  # its outputs end at 65504
    rng = np.random.default_rng(91)
    for G, count in ((1, 1), (8, 16)):
        eng = engine(hkv, G, "e4m3", max_slots=count)
        n = 150
        slots = [eng.acquire() for _ in range(count)]
        for i, s in enumerate(slots):
            k = rows(rng, n, G)
            if i % 2 == 0 and step > 0:
                k[16:32] -= 4  # every second page weighs less, one far less, than its V is large
            eng.rope_append_range(0, s, n, dev(k), dev(far_pages(rng, n, G, step, zero)))
        q = torch.from_numpy((rng.standard_normal((count * n, 4 * G, D)) + 0.5).astype(np.float32)).to(DEV)
        out = window(eng, hkv, slots, [n] * count, q, name).double().cpu().numpy().reshape(count, n, 4 * G, D)
        x = q.to(DT[name]).double().cpu().numpy().reshape(count, n, 4 * G, D)
        for i in range(0, count, 5):
            k, v = cached(eng, hkv, slots[i], n, G)
            h = slice(0, 4) if i % 2 else slice(4 * G - 4, 4 * G)
            g = slice(h.start // 4, h.start // 4 + 1)
            want, bound = weighed(x[i][:, h], k[:, g], v[:, g], 0, name, 7)
            over = np.abs(out[i][:, h] - want) - bound
            assert over.max() <= 0, (G, i, np.unravel_index(over.argmax(), over.shape), over.max())
        eng.close()


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_window_of_values_near_the_largest_floats(hkv_lib, name):
    """V of up to 3e38 over 1,000 rows, split and joined: a mean, not infinity."""
    import hkv
    rng = np.random.default_rng(93)
    eng = engine(hkv, 1, "e4m3")
    s = eng.acquire()
    n = 1000
    v = (rng.uniform(1.0, 3.0, (n, 1, D)) * 1e38).astype(np.float32)
    eng.rope_append_range(0, s, n, dev(rows(rng, n, 1)), dev(v))
    eng.advance([s], 990)
    q = torch.from_numpy(rng.standard_normal((10, 4, D)).astype(np.float32)).to(DEV)
    out = window(eng, hkv, [s], [10], q, name).double().cpu().numpy().reshape(10, 4, D)
    k, v = cached(eng, hkv, s, n, 1)
    want, bound = weighed(q.to(DT[name]).double().cpu().numpy(), k, v, 990, name, 7)
    assert (np.abs(out - want) <= bound).all()
    eng.close()


@pytest.mark.parametrize("cache", ["e4m3", "f16"])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_large_logits(hkv_lib, cache, name):
    """q and K of some 10^4: logits of up to 10^10, apart by far more than one, so that each row is the V of
    one key, whatever its place; and all of them below -2^24 for the keys of one slot."""
    import hkv
    rng = np.random.default_rng(95)
    G, n = 2, 200
    eng = engine(hkv, G, cache)
    q = rng.standard_normal((n, 4 * G, D)).astype(np.float32) * 8000
    for sign in (0, -1):
        s = eng.acquire()
        k = rows(rng, n, G, 0.0) * np.float32(8000)
        if sign:
            k = -np.abs(k)
            q = np.abs(q)
        eng.rope_append_range(0, s, n, dev(k), dev(rows(rng, n, G))) if not sign else \
            eng.qkv_write(0, [s], [n], None, dev(k), dev(rows(rng, n, G)), rotated=True)
        x = torch.from_numpy(q).to(DEV)
        out = window(eng, hkv, [s], [n], x, name).double().cpu().numpy().reshape(n, 4 * G, D)
        kk, vv = cached(eng, hkv, s, n, G)
        x = x.to(DT[name]).double().cpu().numpy()
        sure = 0
        for i in range(n):
            for h in range(4 * G):
                logits = kk[:i + 1, h // 4] @ x[i, h] / np.sqrt(float(D))
                a = np.sort(logits)[::-1]
                # F32 sums of 128 products, q to 2^-17 of its largest value: far less than 2^-14 of sum |q k|
                slack = 2.0 ** -14 * (np.abs(kk[:i + 1, h // 4]) @ np.abs(x[i, h])).max() / np.sqrt(float(D))
                if len(a) == 1 or a[0] - a[1] > 2 * slack + 40:
                    want = vv[np.argmax(logits), h // 4]
                    tol = {"f32": 2.0 ** -20, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[name]
                    assert (np.abs(out[i, h] - want) <= tol * np.abs(want) + 2.0 ** -25).all(), (sign, i, h)
                    sure += 1
        assert sure > n * 4 * G // 2
        eng.release(s)
    eng.close()


@pytest.mark.parametrize("cache", ["e4m3", "f16"])
def test_no_memory_is_taken_inside_a_call(hkv_lib, cache):
    """A new engine's first calls over many rows, the window split over keys, while another stream captures
    (which CUDA refuses every allocation for): they run."""
    import hkv
    rng = np.random.default_rng(97)
    G = 8
    old, new = [3000, 500], [40, 700]

    def calls(eng, slots, data, out, stream=None):
        q, k, v = data
        eng.qkv_write(0, slots, new, q, k, v, q_out=q, stream=stream)
        eng.window_attn(0, slots, new, q, out, stream=stream)
        kk, vv = torch.empty((2, sum(new), G, D), device=DEV).unbind(0) if stream is None else calls.back
        eng.cache_read(0, slots, old, new, kk, vv, dtype=hkv.F32, stream=stream)
        calls.back = (kk, vv)

    results = []
    data = [rng.standard_normal((sum(new), h, D)).astype(np.float32) for h in (4 * G, G, G)]
    kept = [(rows(rng, n, G), rows(rng, n, G)) for n in old]
    for captured in (False, True):
        eng = engine(hkv, G, cache)
        slots = [eng.acquire() for _ in old]
        # one upload of a descriptor, so that the call in question has a buffer to itself: waiting for
        # an upload's event is what CUDA forbids as well while a stream captures
        k, v = (dev(np.concatenate(a)) for a in zip(*kept))
        eng.qkv_write(0, slots, old, None, k, v)
        for s, n in zip(slots, old):
            eng.advance([s], n)
        x = [dev(a) for a in data]
        out = torch.empty((sum(new), 4 * G * D), device=DEV)
        if not captured:
            calls(eng, slots, x, out)
        else:
            work, side = torch.cuda.Stream(), torch.cuda.Stream()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.stream(side):
                graph.capture_begin()
                try:
                    calls(eng, slots, x, out, work.cuda_stream)
                finally:
                    graph.capture_end()
            work.synchronize()
        eng.sync_check()
        results.append(out.clone())
        eng.close()
    assert torch.equal(*results)


@pytest.mark.parametrize("cache", ["e4m3", "f16"])
@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_values_that_are_not_finite_in_long_slots(hkv_lib, cache, name):
    """V that is not finite in some of 1,250 pages, two of them 1,024 apart, in whole and in split tiles: the
    rows that see one have it in its dim, those before it do not."""
    import hkv
    rng = np.random.default_rng(99)
    G, n, t = 1, 19900, 100
    eng = hkv.Engine(n_layers=1, n_head=4, n_head_kv=1, n_pages=1300, max_slots=1, context_length=n + t, device=0,
                     shuffle_seed=9, cache=cache)
    s = eng.acquire()
    k, v = rows(rng, n + t, G), rows(rng, n + t, G)
    bad = {160: 5, 160 + 1024 * 16: 6, 9999: 7, n + 50: 8, n + 99: 9}
    for row, dim in bad.items():
        v[row, 0, dim] = np.nan
    eng.rope_append_range(0, s, n, dev(k[:n]), dev(v[:n]))
    eng.advance([s], n)
    eng.rope_append_range(0, s, t, dev(k[n:]), dev(v[n:]))
    q = torch.from_numpy(rng.standard_normal((t, 4, D)).astype(np.float32)).to(DEV)
    out = window(eng, hkv, [s], [t], q, name).float().cpu().numpy().reshape(t, 4, D)
    want = np.zeros((t, 4, D), bool)
    for row, dim in bad.items():
        want[max(0, row - n):, :, dim] = True
    assert np.array_equal(np.isnan(out), want)
    eng.close()


def test_one_bad_value_does_not_stop_a_prompt(hkv_lib):
    """A prompt of 6,000 with one NaN in V at its start: not all of V is read again for it (the prompt
    took 88 times as long when it was, and takes 6 now; the bound is thirty times)."""
    import hkv
    rng = np.random.default_rng(109)
    G, n = 8, 6000
    eng = engine(hkv, G, "e4m3")
    times = []
    for bad in (False, True):
        s = eng.acquire()
        v = rows(rng, n, G)
        if bad:
            v[3, :, 17] = np.nan
        eng.rope_append_range(0, s, n, dev(rows(rng, n, G)), dev(v))
        q = torch.from_numpy(rng.standard_normal((n, 4 * G, D)).astype(np.float32)).to(DEV).bfloat16()
        out = torch.empty((n, 4 * G * D), dtype=torch.bfloat16, device=DEV)
        best = 1e9
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            eng.window_attn(0, [s], [n], q, out, dtype=hkv.BF16)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        times.append(best)
        got = torch.isnan(out.view(n, 4 * G, D))
        assert got[:, :, 17].sum() == (n - 3) * 4 * G * bad and got.sum() == got[:, :, 17].sum()
        eng.release(s)
    print("ms without and with:", times)
    assert times[1] < 30 * times[0]
    eng.close()


@pytest.mark.parametrize("cache", ["e4m3", "f16"])
def test_f32_windows_keep_22_bits_on_the_average(hkv_lib, cache):
    """The root mean square error of F32 outputs, relative to theirs, against float64 over the cached rows.

    A weight is off, relative to itself, by at most 2^-22 (two F16 parts), by 2^-22 |q| |k| / sqrt(128) through
    q's two parts, and by the 16 cut steps of its logit's sum, each under 2^-23 of a partial sum that is a few
    units at most: 16 * 2^-24 on the average for each unit.  Errors of different keys are independent, as their V
    are: the output's is no more than a weight's, under 2^-17 for partial sums up to 8.  Twice that is the bound.  A
    weight held in one F16 part would be off by 2^-12 / sqrt(3) on the average: nine times the bound."""
    import hkv
    rng = np.random.default_rng(111)
    G = 2
    eng = engine(hkv, G, cache)
    err = size = 0.0
    old, new = [0, 300, 1000], [150, 64, 20]
    slots = [eng.acquire() for _ in old]
    for s, p, n in zip(slots, old, new):
        fill(eng, rng, s, p, G)
        fill(eng, rng, s, n, G, advance=False)
    q = torch.from_numpy(rng.standard_normal((sum(new), 4 * G, D)).astype(np.float32)).to(DEV)
    out = window(eng, hkv, slots, new, q).double().cpu().numpy().reshape(-1, 4 * G, D)
    x = q.double().cpu().numpy()
    at = 0
    for s, p, n in zip(slots, old, new):
        k, v = cached(eng, hkv, s, p + n, G)
        want, _ = weighed(x[at:at + n], k, v, p, "f32", 7)
        err += ((out[at:at + n] - want) ** 2).sum()
        size += (want ** 2).sum()
        at += n
    assert np.sqrt(err / size) < 2.0 ** -16
    eng.close()


@pytest.mark.parametrize("cache", ["e4m3", "f16"])
def test_long_whole_tiles_keep_their_sums(hkv_lib, cache):
    """V = 1 over 30,000 keys in tiles that are not split (19 slots of 8 KV heads): each output is the sum of the
    weights over itself.  The tensor cores cut each of the 16 products of 128 keys by less than a unit in the last
    place of the sum, half of that, 2^-24, on the average; sums leave them every 4 blocks, so no part of one is
    cut more than 64 times: 64 * 2^-24.  The additions outside round to nearest, with no drift: 8 * 2^-24 are
    left for them.  Without the moves the sum drifts by 1.4e-5."""
    import hkv
    rng = np.random.default_rng(113)
    G, n, t, count = 8, 30000, 20, 19
    eng = hkv.Engine(n_layers=1, n_head=32, n_head_kv=G, n_pages=count * 1877, max_slots=count, context_length=n + t,
                     device=0, shuffle_seed=9, cache=cache)
    gen = torch.Generator(device=DEV).manual_seed(113)
    slots = [eng.acquire() for _ in range(count)]
    for s in slots:
        k = torch.randn((n + t, G, D), generator=gen, device=DEV) * 0.3
        v = torch.ones_like(k)
        eng.rope_append_range(0, s, n, k[:n].contiguous(), v[:n].contiguous())
        eng.advance([s], n)
        eng.rope_append_range(0, s, t, k[n:].contiguous(), v[n:].contiguous())
    q = torch.randn((count * t, 32, D), generator=gen, device=DEV)
    out = window(eng, hkv, slots, [t] * count, q).double()
    assert abs((out - 1).mean().item()) < 72 * 2.0 ** -24
    eng.close()


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("old,new", [([700], [300]), ([1500] * 16, [60] * 16)])
def test_window_in_place(hkv_lib, name, old, new):
    """out = q, with equal strides: the same bits as into another tensor, in split and in whole tiles."""
    import hkv
    rng = np.random.default_rng(115)
    G = 8
    eng = engine(hkv, G, "e4m3", n_pages=2000)
    slots = [eng.acquire() for _ in old]
    for s, p, n in zip(slots, old, new):
        fill(eng, rng, s, p, G)
        fill(eng, rng, s, n, G, advance=False)
    q = torch.from_numpy(rng.standard_normal((sum(new), 4 * G, D)).astype(np.float32)).to(DEV)
    out = window(eng, hkv, slots, new, q, name)
    x = q.to(DT[name]).reshape(sum(new), -1)
    eng.window_attn(0, slots, new, x, x, dtype=getattr(hkv, name.upper()))
    eng.sync_check()
    assert torch.equal(out, x)
    eng.close()


def test_window_in_a_capture_is_refused(hkv_lib):
    import hkv
    eng = engine(hkv, 1, "e4m3")
    rng = np.random.default_rng(117)
    s = eng.acquire()
    fill(eng, rng, s, 40, 1, advance=False)
    q = torch.zeros((40, 4 * D), device=DEV)
    out = torch.full_like(q, 5.0)
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        g.capture_begin()
        try:
            with pytest.raises(hkv.HkvError, match="captured") as e:
                eng.window_attn(0, [s], [40], q, out, stream=side.cuda_stream)
            assert e.value.status == hkv.HKV_ERR_INVALID
        finally:
            g.capture_end()
    eng.sync_check()
    assert (out == 5.0).all()
    eng.close()


@pytest.mark.parametrize("cache", ["e4m3", "f16"])
def test_windows_one_after_another(hkv_lib, cache):
    """One engine: a plan found again on another stream (ordered behind the first), small and large split
    windows in turn, two layers, and a slot given back and taken by another request in between."""
    import hkv
    rng = np.random.default_rng(119)
    G = 8
    eng = engine(hkv, G, cache, n_layers=2)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for old, new in (([30], [5]), ([2500, 100], [64, 300]), ([0], [3]), ([4000], [128]), ([17, 300, 900], [1, 90, 2])):
        slots = [eng.acquire() for _ in old]
        for layer in range(2):
            for s, p in zip(slots, old):
                fill(eng, rng, s, p, G, layer, advance=False)
        for s, p in zip(slots, old):
            eng.advance([s], p)
        for layer in range(2):
            for s, n in zip(slots, new):
                fill(eng, rng, s, n, G, layer, advance=False)
        torch.cuda.synchronize()
        q = torch.from_numpy(rng.standard_normal((sum(new), 4 * G, D)).astype(np.float32)).to(DEV)
        outs = torch.zeros((4, sum(new), 4 * G * D), device=DEV)
        for i in range(4):
            streams[i % 2].wait_stream(streams[1 - i % 2])
            eng.window_attn(i // 2, slots, new, q, outs[i], stream=streams[i % 2].cuda_stream)
        for s in streams:
            s.synchronize()
        eng.sync_check()
        for layer in range(2):
            assert torch.equal(outs[2 * layer], outs[2 * layer + 1])
            check(eng, hkv, slots, new, q, outs[2 * layer], "f32", layer)
        for s in slots:
            eng.release(s)
    eng.close()


@pytest.mark.parametrize("low,high", [(0.0, 1e12), (0.0, 1e30), (1e-25, 1e20), (1e25, 0.0)])
@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_window_where_v_jumps_between_blocks(hkv_lib, name, low, high):
    """Whole blocks of keys whose V is far below, or above, that of the next ones, at like weights: the sum of
    weights keeps both, in whole tiles (19 slots of 8 heads) and in split ones."""
    import hkv
    rng = np.random.default_rng(121)
    n, t = 640, 20
    for G, count in ((1, 1), (8, 19)):
        eng = engine(hkv, G, "e4m3", max_slots=count)
        slots = [eng.acquire() for _ in range(count)]
        for s in slots:
            v = rows(rng, n + t, G)
            v[:256] *= np.float32(low)
            v[256:] *= np.float32(high)
            k = rows(rng, n + t, G) * np.float32(0.3)
            eng.rope_append_range(0, s, n, dev(k[:n]), dev(v[:n]))
            eng.advance([s], n)
            eng.rope_append_range(0, s, t, dev(k[n:]), dev(v[n:]))
        q = torch.from_numpy(rng.standard_normal((count * t, 4 * G, D)).astype(np.float32)).to(DEV)
        out = window(eng, hkv, slots, [t] * count, q, name).double().cpu().numpy().reshape(count, t, 4 * G, D)
        x = q.to(DT[name]).double().cpu().numpy().reshape(count, t, 4 * G, D)
        for i in range(0, count, 9):
            k, v = cached(eng, hkv, slots[i], n + t, G)
            want, bound = weighed(x[i][:, :4], k[:, :1], v[:, :1], n, name, 7)
            over = np.abs(out[i][:, :4] - want) - bound
            assert over.max() <= 0, (G, i, np.unravel_index(over.argmax(), over.shape), over.max())
        eng.close()
