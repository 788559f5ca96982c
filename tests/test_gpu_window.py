"""hkv_window_attn on the GPU: several new tokens per slot over the paged cache.

Held to a float64 attention over the rows the cache holds (read back exactly), so
the bound covers the attention alone.
"""
from __future__ import annotations

import numpy as np
import pytest

from cache8_model import D, attention, attention_tolerance
from test_gpu_cache8 import DEV, cache8, dev, rows  # noqa: F401 (fixture)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def tolerance(name, big, n_rows, vmax, want, q, k):
    """F32: attention_tolerance().  F16 and BF16: the weights are rounded to F16 (2^-11
    relative, on top of the F32 path's) and the output once to its type; F16 outputs
    below 2^-14 have steps of 2^-24.  F16 q enters exactly.  BF16 q (8 bits) enters as two
    E4M3 numbers of 4 bits, scaled so that the row's largest value is at least 224: exact
    down to 2^-2 (the second part is a multiple of 2^-9), off by at most 2^-10 below that, which
    is 2^-10 / 224 of the row's largest value for each dim, and moves every weight by twice that."""
    t = attention_tolerance(big, n_rows, vmax)
    if name == "f32":
        return t
    t += vmax * 2.0 ** -11
    if name == "bf16":
        t += 2 * vmax * np.abs(q).max() * 2.0 ** -10 / 224 * np.abs(k).sum(-1).max() / np.sqrt(128.0)
    return t + HALF[name] * (np.abs(want) + t) + (2.0 ** -25 if name == "f16" else 0.0)


def window(eng, hkv, slots, new, q, name="f32", layer=0, **kw):
    out = torch.full((q.shape[0] + 1, q.shape[1] * D), 5.0, dtype=DT[name], device=DEV)
    eng.window_attn(layer, slots, new, q.to(DT[name]), out, dtype=getattr(hkv, name.upper()), **kw)
    eng.sync_check()
    assert (out[-1] == 5.0).all()  # rows behind the last, as they were
    return out[:-1]


def check(eng, hkv, slots, new, q, out, name, layer=0):
    """Every row of `out` against float64 over the rows that the cache holds."""
    H = q.shape[1]
    q64 = q.to(DT[name]).double().cpu().numpy()
    got = out.double().cpu().numpy().reshape(-1, H, D)
    at = 0
    for s, n in zip(slots, new):
        if not n:
            continue
        p = eng.length(s)
        k, v = torch.empty((2, p + n, H // 4, D), device=DEV).unbind(0)
        eng.cache_read(layer, [s], [0], [p + n], k, v, dtype=hkv.F32)
        torch.cuda.synchronize()
        k, v = k.cpu().numpy(), v.cpu().numpy()
        want, big = attention(q64[at:at + n], k, v, p)
        tol = tolerance(name, big, p + n, np.abs(v).max(), want, q64[at:at + n], k)
        over = float((np.abs(got[at:at + n] - want) - tol).max())
        assert over <= 0, (s, p, n, over, float(np.abs(got[at:at + n] - want).max()))
        at += n


def engine(hkv, G, cache, n_pages=1024, max_slots=16, n_layers=1):
    return hkv.Engine(n_layers=n_layers, n_head=4 * G, n_head_kv=G, n_pages=n_pages, max_slots=max_slots,
                      context_length=16384, device=0, shuffle_seed=9, cache=cache)


def fill(eng, rng, slot, n, G, layer=0, advance=True, scale=1.0):
    if n:
        eng.rope_append_range(layer, slot, n, dev(rows(rng, n, G)), dev(rows(rng, n, G) * np.float32(scale)))
        if advance:
            eng.advance([slot], n)


@pytest.mark.parametrize("cache", ["e4m3", "f16"])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("G,old,new", [
    (8, [0], [1]), (8, [0], [16]), (2, [0], [63]), (2, [0], [64]), (2, [0], [65]), (1, [0], [130]),
    (8, [770], [37]), (4, [15, 16, 17, 0], [1, 2, 3, 4]), (2, [100, 0, 255, 31], [64, 0, 200, 1]),
    (1, [3000], [5]), (1, [127], [1]), (1, [128], [1]), (1, [0], [700]), (2, [5000, 10], [3, 400])])
def test_window_against_float64(hkv_lib, cache, name, G, old, new):
    import hkv
    rng = np.random.default_rng(sum(old) + 7 * sum(new))
    eng = engine(hkv, G, cache)
    slots = [eng.acquire() for _ in old]
    for s, p, n in zip(slots, old, new):
        fill(eng, rng, s, p, G)
        fill(eng, rng, s, n, G, advance=False)
    q = torch.from_numpy(rng.standard_normal((sum(new), 4 * G, D)).astype(np.float32) * 2).to(DEV)
    out = window(eng, hkv, slots, new, q, name)
    check(eng, hkv, slots, new, q, out, name)
    assert torch.equal(out, window(eng, hkv, slots, new, q, name))  # the same bits again
    eng.close()


def test_window_strides(hkv_lib):
    import hkv
    rng = np.random.default_rng(5)
    G, H = 2, 8
    eng = engine(hkv, G, "e4m3")
    s = eng.acquire()
    fill(eng, rng, s, 50, G)
    fill(eng, rng, s, 70, G, advance=False)
    for name in ("f32", "bf16"):
        x = torch.from_numpy(rng.standard_normal((70, H * D + 64)).astype(np.float32)).to(DEV, DT[name])
        out = torch.full((70, H * D + 32), 5.0, dtype=DT[name], device=DEV)
        eng.window_attn(0, [s], [70], x, out, dtype=getattr(hkv, name.upper()), q_stride=x.stride(0),
                        out_stride=out.stride(0))
        eng.sync_check()
        assert (out[:, H * D:] == 5.0).all()
        q = x[:, :H * D].reshape(70, H, D).float()
        check(eng, hkv, [s], [70], q, out[:, :H * D].contiguous(), name)
    eng.close()


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_window_exponents_far_apart(hkv_lib, name):
    """V pages 2^5 apart each (2^60 over the slot, rising and falling), K pages 2^-11 apart."""
    import hkv
    rng = np.random.default_rng(15)
    G = 1
    eng = engine(hkv, G, "e4m3")
    for flip in (1, -1):
        s = eng.acquire()
        k, v = rows(rng, 200, G), rows(rng, 200, G)
        for p in range(13):
            v[16 * p:16 * p + 16] *= 2.0 ** (flip * 5 * (p - 6))
            k[16 * p:16 * p + 16] *= 2.0 ** -(p % 12)
        eng.rope_append_range(0, s, 200, dev(k), dev(v))
        q = torch.from_numpy(rng.standard_normal((200, 4, D)).astype(np.float32)).to(DEV)
        out = window(eng, hkv, [s], [200], q, name)
        # row by row, so that the bound goes by the V that the row sees
        kk, vv = torch.empty((2, 200, G, D), device=DEV).unbind(0)
        eng.cache_read(0, [s], [0], [200], kk, vv, dtype=hkv.F32)
        kk, vv = kk.cpu().numpy(), vv.cpu().numpy()
        q64 = q.to(DT[name]).double().cpu().numpy()
        got = out.double().cpu().numpy().reshape(200, 4, D)
        for i in range(0, 200, 3):
            want, big = attention(q64[i:i + 1], kk[:i + 1], vv[:i + 1], i)
            tol = tolerance(name, big, i + 1, np.abs(vv[:i + 1]).max(), want, q64[i], kk[:i + 1])
            assert float((np.abs(got[i] - want[0]) - tol).max()) <= 0, i
    eng.close()


@pytest.mark.parametrize("cache", ["e4m3", "f16"])
def test_window_ignores_what_it_must_not_see(hkv_lib, cache):
    """Pages that held NaN and huge rows of another request; large logits (one key takes all)."""
    import hkv
    rng = np.random.default_rng(25)
    G = 2
    eng = engine(hkv, G, cache, n_pages=20)
    s = eng.acquire()
    bad = np.full((320, G, D), np.nan, np.float32)
    bad[::3] = np.inf
    eng.rope_append_range(0, s, 320, dev(bad), dev(bad))
    eng.release(s)
    slots = [eng.acquire(), eng.acquire()]
    fill(eng, rng, slots[0], 21, G)
    fill(eng, rng, slots[0], 80, G, advance=False)
    fill(eng, rng, slots[1], 7, G, advance=False)
    q = torch.from_numpy(rng.standard_normal((87, 8, D)).astype(np.float32) * 30).to(DEV)
    for name in ("f32", "f16", "bf16"):
        out = window(eng, hkv, slots, [80, 7], q, name)
        assert torch.isfinite(out).all()
        check(eng, hkv, slots, [80, 7], q, out, name)
    eng.close()


@pytest.mark.parametrize("cache", ["e4m3", "f16"])
def test_long_f32_sums_keep_their_bits(hkv_lib, cache):
    """V = 1 everywhere: each output is the sum of the weights over itself.  The tensor cores cut each
    of the 16 products of 128 keys by up to an ulp of the sum (at most 2^-23 of it, half of that on
    average); over 30,000 keys added up there this would come to 1.4e-5.  With the sums moved out after
    8 blocks at most 8 * 16 cuts act on any part of it: 128 * 2^-24 on average, and one rounding to F32
    (2^-24) for each of the 30 moves and, of l, a few per block at random."""
    import hkv
    rng = np.random.default_rng(28)
    n, t = 28000, 2100
    eng = hkv.Engine(n_layers=1, n_head=4, n_head_kv=1, n_pages=2000, max_slots=1, context_length=n + t, device=0,
                     shuffle_seed=9, cache=cache)
    s = eng.acquire()
    k = torch.from_numpy((rng.standard_normal((n + t, 1, D)) * 0.3).astype(np.float32)).to(DEV)
    v = torch.ones_like(k)
    eng.rope_append_range(0, s, n, k[:n].contiguous(), v[:n].contiguous())
    eng.advance([s], n)
    eng.rope_append_range(0, s, t, k[n:].contiguous(), v[n:].contiguous())
    q = torch.from_numpy(rng.standard_normal((t, 4, D)).astype(np.float32)).to(DEV)
    out = window(eng, hkv, [s], [t], q, "f32").double()
    assert abs((out - 1).mean().item()) < 128 * 2.0 ** -24 + 31 * 2.0 ** -24
    eng.close()


@pytest.mark.parametrize("cache,rise,v_step", [
    ("e4m3", 10.0, 0), ("e4m3", -10.0, 0), ("e4m3", 0.0, 3), ("e4m3", 0.0, -3), ("e4m3", 4.0, 3), ("f16", 10.0, 0),
    ("f16", 4.0, 1)])
@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_long_tiles_whose_bounds_move(hkv_lib, cache, rise, v_step, name):
    """Sixteen slots of 8 KV heads, so that no tile is split: 17 blocks of keys whose logits rise or fall
    by up to 163 bits over the slot, and V pages whose sizes do, by 2^51: what is summed first has to be
    held in other units many times, and to vanish in the end."""
    import hkv
    rng = np.random.default_rng(29)
    G, n = 8, 2100
    eng = engine(hkv, G, cache, n_pages=16 * 134)
    dirs = rng.choice([-1.0, 1.0], (1, G, D)).astype(np.float32)
    new = [20] * 15 + [64]
    slots = [eng.acquire() for _ in new]
    for s, t in zip(slots, new):
        at = np.arange(n + t, dtype=np.float32) / n
        k = dirs * (rise * (at - 0.5))[:, None, None] + 0.05 * rows(rng, n + t, G)
        v = rows(rng, n + t, G) * np.exp2(v_step * (np.arange(n + t) // 128 - 8)).astype(np.float32)[:, None, None]
        for r0, r1 in ((0, n), (n, n + t)):
            eng.qkv_write(0, [s], [r1 - r0], None, dev(k[r0:r1]), dev(v[r0:r1]), rotated=True)
            if r0 == 0:
                eng.advance([s], n)
    q = np.repeat(dirs, sum(new), 0).repeat(4, 1) + 0.3 * rng.standard_normal((sum(new), 4 * G, D)).astype(np.float32)
    q = torch.from_numpy(q.astype(np.float32)).to(DEV)
    out = window(eng, hkv, slots, new, q, name)
    check(eng, hkv, slots, new, q, out, name)
    assert torch.equal(out, window(eng, hkv, slots, new, q, name))
    eng.close()


@pytest.mark.parametrize("cache", ["e4m3", "f16"])
@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_window_rows_before_a_value_that_is_not_finite(hkv_lib, cache, name):
    """A NaN in one dim of V at position 40 (and inf, -inf in an F16 cache): rows before it do not
    know of it, rows from it on have it in that dim and KV head alone."""
    import hkv
    rng = np.random.default_rng(27)
    G = 2
    eng = engine(hkv, G, cache)
    s = eng.acquire()
    fill(eng, rng, s, 10, G)
    k, v = rows(rng, 90, G), rows(rng, 90, G)
    v[30, 1, 77] = np.nan
    if cache == "f16":
        v[60, 0, 3], v[61, 0, 100] = np.inf, -np.inf
    eng.rope_append_range(0, s, 90, dev(k), dev(v))
    q = torch.from_numpy(rng.standard_normal((90, 8, D)).astype(np.float32)).to(DEV)
    out = window(eng, hkv, [s], [90], q, name).float().cpu().numpy().reshape(90, 8, D)
    want = np.zeros((90, 8, D), bool)
    want[30:, 4:, 77] = True
    assert np.array_equal(np.isnan(out), want)
    if cache == "f16":
        want[:] = False
        want[60:, :4, 3] = want[61:, :4, 100] = True
        assert np.array_equal(np.isinf(out), want)
        assert (out[60:, :4, 3] > 0).all() and (out[61:, :4, 100] < 0).all()
    k[50, 0, 5] = np.nan  # in K: the rows that see it, of that KV head
    eng.rope_append_range(0, s, 90, dev(k), dev(np.nan_to_num(v, nan=1.0, posinf=1.0, neginf=1.0)))
    out = window(eng, hkv, [s], [90], q, name).float().cpu().numpy().reshape(90, 8, D)
    want[:] = False
    want[50:, :4] = True
    assert np.array_equal(np.isnan(out), want)
    eng.close()


@pytest.mark.parametrize("cache,n_pages", [("e4m3", 140000), ("f16", 72000)])
def test_pools_beyond_32_bit_offsets(hkv_lib, cache, n_pages):
    """Layers of 4.6 GB, pages scattered over them: writes, reads, windows and a decode step in the
    second layer (bytes 4.6e9 to 9.2e9 of the pool)."""
    import hkv
    rng = np.random.default_rng(30)
    G = 8
    eng = hkv.Engine(n_layers=2, n_head=4 * G, n_head_kv=G, n_pages=n_pages, max_slots=4, context_length=4096, device=0,
                     shuffle_seed=31, cache=cache)
    old, new = [300, 17, 0], [70, 64, 33]
    slots = [eng.acquire() for _ in old]
    for s, p, n in zip(slots, old, new):
        fill(eng, rng, s, p, G, layer=1)
        fill(eng, rng, s, n, G, layer=1, advance=False)
    assert max(max(eng.pages(s)) for s in slots) > n_pages // 2
    q = torch.from_numpy(rng.standard_normal((sum(new), 4 * G, D)).astype(np.float32)).to(DEV)
    for name in ("f32", "bf16"):
        check(eng, hkv, slots, new, q, window(eng, hkv, slots, new, q, name, layer=1), name, layer=1)
    for s, n in zip(slots, new):
        eng.advance([s], n)
    # one token more: the decode step's output is the window's over the row it wrote
    x, k, v = (torch.from_numpy(rng.standard_normal((3, h, D)).astype(np.float32)).to(DEV) for h in (4 * G, G, G))
    step = torch.empty((3, 4 * G * D), device=DEV)
    eng.decode_step(1, slots, x, k, v, step)
    turned = torch.empty_like(x)
    eng.qkv_write(1, slots, [1] * 3, x, k, v, q_out=turned)
    one = window(eng, hkv, slots, [1] * 3, turned, layer=1)
    check(eng, hkv, slots, [1] * 3, turned, one, "f32", layer=1)
    check(eng, hkv, slots, [1] * 3, turned, step, "f32", layer=1)
    eng.close()


@pytest.mark.parametrize("cache", ["e4m3", "f16"])
def test_one_token_window_is_the_decode(hkv_lib, oracle, rope_tables, cache):
    """n_tokens = 1 against hkv_decode_attn on the same cache (both F32 paths)."""
    import hkv
    rng = np.random.default_rng(35)
    G = 8
    cos, sin = rope_tables
    eng = engine(hkv, G, cache)
    lens = [0, 5, 16, 300, 2000]
    slots = [eng.acquire() for _ in lens]
    for s, n in zip(slots, lens):
        fill(eng, rng, s, n, G)
    k, v = dev(rows(rng, 5, G)), dev(rows(rng, 5, G))
    q = rng.standard_normal((5, 32, D)).astype(np.float32)
    a = torch.empty((5, 32 * D), device=DEV)
    eng.decode_step(0, slots, dev(q), k, v, a)
    qr = np.stack([oracle.rope_neox(q[i], cos[n], sin[n]) for i, n in enumerate(lens)])
    b = window(eng, hkv, slots, [1] * 5, dev(qr))
    check(eng, hkv, slots, [1] * 5, dev(qr), b, "f32")
    check(eng, hkv, slots, [1] * 5, dev(qr), a, "f32")
    eng.close()


@pytest.mark.parametrize("cache", ["e4m3", "f16"])
def test_prompt_then_decode(hkv_lib, cache):
    """The operators in a row, as a request uses them: qkv_write and window_attn over a prompt in two
    chunks and two layers, then decode steps, against one float64 pass over all rows."""
    import hkv
    rng = np.random.default_rng(45)
    G, H, T = 2, 8, 150
    eng = engine(hkv, G, cache, n_layers=2)
    s = eng.acquire(T + 4)
    x = torch.from_numpy(rng.standard_normal((2, T, (H + 2 * G) * D)).astype(np.float32)).to(DEV)
    qn, kn = dev(rng.random(D) + 0.5), dev(rng.random(D) + 0.5)
    st = x.stride(1)
    at = 0
    for n in (97, 53):
        for layer in range(2):
            rows_ = x[layer, at:at + n]
            q = torch.empty((n, H, D), device=DEV)
            eng.qkv_write(layer, [s], [n], rows_, rows_[:, H * D:], rows_[:, (H + G) * D:], q_norm=qn, k_norm=kn,
                          q_out=q, q_stride=st, k_stride=st, v_stride=st)
            out = window(eng, hkv, [s], [n], q, layer=layer)
            check(eng, hkv, [s], [n], q, out, "f32", layer)
        eng.advance([s], n)
        at += n
    for step in range(3):
        for layer in range(2):
            q = rng.standard_normal((1, H, D)).astype(np.float32)
            out = torch.empty((1, H * D), device=DEV)
            eng.decode_step(layer, [s], dev(q), dev(rows(rng, 1, G)), dev(rows(rng, 1, G)), out)
            cos, sin = (t[eng.length(s)].astype(np.float64) for t in eng.rope_tables())
            a, b = q[..., :64].astype(np.float64), q[..., 64:].astype(np.float64)
            qr = np.concatenate([a * cos - b * sin, a * sin + b * cos], -1)
            check(eng, hkv, [s], [1], torch.from_numpy(qr.astype(np.float32)).to(DEV), out, "f32", layer)
        eng.advance([s], 1)
    eng.sync_check()
    eng.close()
