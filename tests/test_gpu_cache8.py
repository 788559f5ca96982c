"""The 8-bit cache on the GPU: writes, read back, decode attention.

Cells are held to the format's definition bit for bit (cache8_model.py), decode
attention to a float64 attention over those cells within the bound that
attention_tolerance() derives.
"""
from __future__ import annotations

import numpy as np
import pytest

from cache8_model import D, PAGE, SlotModel, attention, attention_tolerance, round_e4m3

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(DEV)


class Cache8:
    """An E4M3 engine of one layer or more and the model of every slot."""

    def __init__(self, hkv, oracle, tables, G=8, n_layers=1, n_pages=512, max_slots=40, context=33000, seed=5):
        self.hkv, self.o, self.G, self.H = hkv, oracle, G, 4 * G
        self.cos, self.sin = tables
        self.L = n_layers
        self.eng = hkv.Engine(n_layers=n_layers, n_head=4 * G, n_head_kv=G, n_pages=n_pages, max_slots=max_slots,
                              context_length=min(context, 32768), device=0, shuffle_seed=seed, cache="e4m3")
        self.k, self.v = {}, {}

    def slot(self, capacity=0):
        s = self.eng.acquire(capacity)
        self.k[s] = [SlotModel(self.G) for _ in range(self.L)]
        self.v[s] = [SlotModel(self.G) for _ in range(self.L)]
        return s

    def rope(self, x, pos):
        """F32 rows [n][heads][D] rotated at positions pos, as the oracle rounds."""
        return np.stack([self.o.rope_neox(np.ascontiguousarray(r), self.cos[p], self.sin[p])
                         for r, p in zip(x, pos)]) if len(x) else x

    def model_write(self, s, k, v, layer=0, roped=False):
        p = self.eng.length(s)
        self.k[s][layer].write(p, k if roped else self.rope(k, range(p, p + len(k))))
        self.v[s][layer].write(p, v)

    def prefill(self, s, k, v, layer=0, advance=True):
        if len(k):
            self.eng.rope_append_range(layer, s, len(k), dev(k), dev(v))
            self.model_write(s, k, v, layer)
            if advance:
                self.eng.advance([s], len(k))

    def read(self, s, pos0, n, layer=0, dtype=torch.float32):
        k = torch.empty((n, self.G, D), dtype=dtype, device=DEV)
        v = torch.empty_like(k)
        self.eng.cache_read(layer, [s], [pos0], [n], k, v, dtype=self.hkv.F32 if dtype == torch.float32 else self.hkv.F16)
        torch.cuda.synchronize()
        return k.cpu().numpy(), v.cpu().numpy()

    def check(self, s, n=None, layer=0):
        """Rows [0, n) of the slot equal the model's, every bit (NaN for NaN)."""
        n = self.eng.length(s) if n is None else n
        k, v = self.read(s, 0, n, layer)
        for got, want, name in ((k, self.k[s][layer].values[:n], "k"), (v, self.v[s][layer].values[:n], "v")):
            with np.errstate(over="ignore"):
                want = want.astype(np.float32)
            bad = ~((got == want) | (np.isnan(got) & np.isnan(want)))
            assert not bad.any(), (name, np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])

    def check_attention(self, slots, q, out, layer=0):
        out = out.cpu().numpy().reshape(len(slots), self.H, D)
        for i, s in enumerate(slots):
            p = self.eng.length(s)
            k, v = self.k[s][layer].values[:p + 1], self.v[s][layer].values[:p + 1]
            want, big = attention(self.rope(q[i:i + 1], [p]), k, v, p)
            tol = attention_tolerance(big, p + 1, np.abs(v).max())
            err = np.abs(out[i] - want[0]).max()
            assert err <= tol, (i, p, err, tol)

    def close(self):
        self.eng.sync_check()
        self.eng.close()


@pytest.fixture
def cache8(hkv_lib, oracle, rope_tables):
    import hkv
    made = []

    def make(**kw):
        made.append(Cache8(hkv, oracle, rope_tables, **kw))
        return made[-1]

    yield make
    for c in made:
        c.close()


def rows(rng, n, G, spread=0.5):
    return (rng.standard_normal((n, G, D)) * np.exp(spread * rng.standard_normal((n, 1, 1)))).astype(np.float32)


@pytest.mark.parametrize("G", [1, 2, 8])
@pytest.mark.parametrize("chunks", [[1] * 20, [15, 1, 1, 16, 3], [33, 100], [5, 1, 27, 1, 1, 64]])
def test_range_and_single_writes_are_the_definition(cache8, G, chunks):
    rng = np.random.default_rng(G * 100 + len(chunks))
    c = cache8(G=G)
    s = c.slot()
    for i, n in enumerate(chunks):
        k, v = rows(rng, n, G), rows(rng, n, G)
        if n == 1 and i % 2:
            c.eng.rope_append(0, [s], dev(k), dev(v))
            c.model_write(s, k, v)
            c.eng.advance([s], 1)
        else:
            c.prefill(s, k, v)
    c.check(s)
    # the F16 view rounds those values once
    n = c.eng.length(s)
    kh, vh = torch.empty((2, n, G, D), dtype=torch.int16, device=DEV).unbind(0)
    c.eng.gather(s, 0, 0, n, kh, vh)
    k16, v16 = c.read(s, 0, n, dtype=torch.float16)
    assert np.array_equal(kh.cpu().numpy().view(np.float16), k16)
    assert np.array_equal(v16, c.v[s][0].values[:n].astype(np.float16))


def test_raw_append_and_growing_rows(cache8):
    """Each row 2 to 5 times the one before: every append rounds the page again."""
    rng = np.random.default_rng(7)
    c = cache8(G=2)
    s = c.slot()
    for r in range(40):
        g = 10.0 ** (-20 + r)
        k, v = (rng.standard_normal((1, 2, D)) * g).astype(np.float32), (rng.standard_normal((1, 2, D)) / g).astype(np.float32)
        c.eng.append(0, [s], dev(k), dev(v))
        c.model_write(s, k, v, roped=True)
        c.eng.advance([s], 1)
        c.check(s)


def test_special_values(cache8):
    """Zeros, signed zeros, subnormals, the borders of the exponent rule, the largest
    floats, and values that are not finite next to finite ones."""
    c = cache8(G=1)
    s = c.slot()
    base = np.zeros((16, 1, D), np.float32)
    rng = np.random.default_rng(3)
    for fill in ("zero", "subnormal", "border", "above", "huge", "inf", "nan", "allnan", "ties"):
        k, v = base.copy(), base.copy()
        if fill == "subnormal":
            v[:, 0, :] = 1e-41
            v[3, 0, 5] = -1e-45
        elif fill == "border":
            v[2, 0, 7], v[1, 0, 1] = 448 * 2.0 ** -9, -3 * 2.0 ** -9
        elif fill == "above":
            v[2, 0, 7], v[1, 0, 1] = np.nextafter(np.float32(448 * 2.0 ** -9), np.float32(9)), 448 * 2.0 ** -9
        elif fill == "huge":
            v[0, 0, 0], v[1, 0, 1], v[2, 0, 2] = np.finfo(np.float32).max, -3e38, 1.0
        elif fill in ("inf", "nan"):
            v[:] = rng.standard_normal(v.shape)
            v[4, 0, 9] = np.inf if fill == "inf" else np.nan
            v[5, 0, 0] = -np.inf
        elif fill == "allnan":
            v[:] = np.nan
        elif fill == "ties":
            v[0, 0, :] = (16 + np.arange(D) % 16 + 0.5) * np.where(np.arange(D) % 2, 1, -1)
            v[1, 0, 0] = 448
            v[2, 0, :] = np.arange(D) * 2.0 ** -10
        elif fill == "zero":
            v[0, 0, 0] = -0.0
        c.eng.advance([s], 0)
        c.prefill(s, k, v)
        c.check(s)


def test_first_row_of_a_page_starts_it_anew(cache8):
    """A page taken back after a rollback, or rewritten from its first row, holds no trace
    of the larger rows it had; a rewrite inside a page keeps its exponent."""
    rng = np.random.default_rng(11)
    c = cache8(G=2)
    s = c.slot()
    c.prefill(s, rows(rng, 20, 2) * 1e6, rows(rng, 20, 2) * 1e6)
    c.eng.set_length(s, 0)
    k, v = rows(rng, 9, 2), rows(rng, 9, 2)
    c.k[s], c.v[s] = [SlotModel(2)], [SlotModel(2)]
    c.prefill(s, k, v)
    c.check(s)
    c.eng.set_length(s, 5)
    k, v = rows(rng, 30, 2) * 0.01, rows(rng, 30, 2) * 50
    c.prefill(s, k, v)
    c.check(s)


@pytest.mark.parametrize("G", [1, 4, 8])
@pytest.mark.parametrize("fused", [False, True])
def test_decode_over_ragged_lengths(cache8, G, fused):
    rng = np.random.default_rng(G)
    c = cache8(G=G, n_pages=1200)
    lens = [0, 1, 14, 15, 16, 17, 30, 31, 33, 255, 256, 1000, 4095]
    slots = [c.slot(n + 3) for n in lens]
    for s, n in zip(slots, lens):
        c.prefill(s, rows(rng, n, G), rows(rng, n, G))
    for step in range(2):
        n = len(slots)
        q, k, v = rng.standard_normal((n, 4 * G, D)).astype(np.float32), rows(rng, n, G, 1.0), rows(rng, n, G, 1.0)
        out = torch.empty((n, 4 * G * D), device=DEV)
        if fused:
            c.eng.decode_step(0, slots, dev(q), dev(k), dev(v), out)
        else:
            c.eng.rope_append(0, slots, dev(k), dev(v))
            c.eng.decode_attn(0, slots, dev(q), out)
        for i, s in enumerate(slots):
            c.model_write(s, k[i:i + 1], v[i:i + 1])
        c.check_attention(slots, q, out)
        c.eng.advance(slots, 1)
        for s in slots[:8]:
            c.check(s)
        slots = slots[::-1]


@pytest.mark.parametrize("seed,n,hi", [(7, 16, 4096), (1, 32, 2048), (2, 15, 2000), (3, 20, 8000)])
def test_decode_over_batches_of_unequal_lengths(cache8, seed, n, hi):
    """Segments of more than 16 partials among shorter ones (the combine launch), and of more than 32
    (two levels in the launch): the fused step and the separate calls agree bit for bit, and every third
    slot is within the bound of float64."""
    rng = np.random.default_rng(seed)
    lens = [hi] + [int(x) for x in rng.integers(1, hi, n - 1)]
    c = cache8(G=8, n_pages=sum(x // PAGE + 2 for x in lens), max_slots=n, context=hi + 32)
    slots = [c.slot() for _ in lens]
    for s, t in zip(slots, lens):
        c.eng.rope_append_range(0, s, t, dev(rows(rng, t, 8)), dev(rows(rng, t, 8)))
        c.eng.advance([s], t)
    q, k, v = (rng.standard_normal((n, h, D)).astype(np.float32) for h in (32, 8, 8))
    out, again = torch.zeros((2, n, 32 * D), device=DEV).unbind(0)
    c.eng.rope_append(0, slots, dev(k), dev(v))
    c.eng.decode_attn(0, slots, dev(q), out)
    c.eng.decode_step(0, slots, dev(q), dev(k), dev(v), again)
    c.eng.sync_check()
    assert torch.equal(out, again)
    q_rot = torch.empty((n, 32, D), device=DEV)
    kk, vv = torch.empty((2, max(lens) + 1, 8, D), device=DEV).unbind(0)
    import hkv
    c.eng.qkv_write(0, slots, [1] * n, dev(q), dev(k), dev(v), q_out=q_rot)
    for e in range(0, n, 3):
        t = lens[e] + 1
        c.eng.cache_read(0, [slots[e]], [0], [t], kk, vv, dtype=hkv.F32)
        torch.cuda.synchronize()
        k64, v64 = kk[:t].cpu().numpy(), vv[:t].cpu().numpy()
        want, big = attention(q_rot[e:e + 1].double().cpu().numpy(), k64, v64, t - 1)
        got = out[e].double().cpu().numpy().reshape(1, 32, D)
        assert float(np.abs(got - want).max()) <= attention_tolerance(big, t, np.abs(v64).max()), e


@pytest.mark.parametrize("G,length", [(8, 1100), (8, 1500), (8, 32767), (1, 32767), (2, 5000), (1, 17)])
def test_decode_of_one_request(cache8, G, length):
    """One request alone: its segments go through clusters, the combine launch or groups."""
    rng = np.random.default_rng(length)
    c = cache8(G=G, n_pages=2100, max_slots=2)
    s = c.slot(length + 1)
    c.prefill(s, rows(rng, length, G), rows(rng, length, G))
    q, k, v = rng.standard_normal((1, 4 * G, D)).astype(np.float32), rows(rng, 1, G), rows(rng, 1, G)
    out = torch.empty((1, 4 * G * D), device=DEV)
    c.eng.decode_step(0, [s], dev(q), dev(k), dev(v), out)
    c.model_write(s, k, v)
    c.check_attention([s], q, out)
    again = torch.empty_like(out)
    c.eng.decode_attn(0, [s], dev(q), again)
    assert torch.equal(out, again)


def test_fused_step_and_separate_calls_agree(cache8):
    rng = np.random.default_rng(23)
    outs, cells = [], []
    lens = [5, 16, 47, 300, 1111]
    data = [(rows(rng, n, 8), rows(rng, n, 8)) for n in lens]
    steps = [(rng.standard_normal((5, 32, D)).astype(np.float32), rows(rng, 5, 8, 1.5), rows(rng, 5, 8, 1.5)) for _ in range(12)]
    for fused in (True, False):
        c = cache8(G=8)
        slots = [c.slot() for _ in lens]
        for s, (k, v) in zip(slots, data):
            c.prefill(s, k, v)
        for q, k, v in steps:
            out = torch.empty((5, 32 * D), device=DEV)
            if fused:
                c.eng.decode_step(0, slots, dev(q), dev(k), dev(v), out)
            else:
                c.eng.rope_append(0, slots, dev(k), dev(v))
                c.eng.decode_attn(0, slots, dev(q), out)
            c.eng.advance(slots, 1)
            outs.append(out.cpu())
        cells.append([c.read(s, 0, c.eng.length(s)) for s in slots])
    for a, b in zip(outs[:12], outs[12:]):
        assert torch.equal(a, b)
    for a, b in zip(*cells):
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_exponents_far_apart_between_pages(cache8):
    """V of neighbouring pages 2^60 apart either way, K 2^12 apart: the output keeps the
    accuracy of the pages that weigh in it."""
    rng = np.random.default_rng(31)
    c = cache8(G=2)
    s, t = c.slot(), c.slot()
    for slot, flip in ((s, 1), (t, -1)):
        k, v = rows(rng, 200, 2), rows(rng, 200, 2)
        for p in range(13):
            sl = slice(16 * p, 16 * p + 16)
            v[sl] *= 2.0 ** (flip * 5 * (p - 6))
            k[sl] *= 2.0 ** -(p % 12)
        c.prefill(slot, k, v)
    q, k, v = rng.standard_normal((2, 8, D)).astype(np.float32), rows(rng, 2, 2), rows(rng, 2, 2)
    out = torch.empty((2, 8 * D), device=DEV)
    c.eng.decode_step(0, [s, t], dev(q), dev(k), dev(v), out)
    for i, x in enumerate((s, t)):
        c.model_write(x, k[i:i + 1], v[i:i + 1])
    c.check_attention([s, t], q, out)
    # all weight on a page of small V while a page of large V has none
    u = c.slot()
    k, v = np.zeros((48, 2, D), np.float32), rows(rng, 48, 2)
    k[16:32, :, :] = 4.0
    v[16:32] *= 2.0 ** -40
    c.eng.advance([u], 0)
    for r in range(48):  # raw rows: no rotation, so that q . k is the same for a page
        c.eng.append(0, [u], dev(k[r:r + 1]), dev(v[r:r + 1]))
        c.model_write(u, k[r:r + 1], v[r:r + 1], roped=True)
        c.eng.advance([u], 1)
    c.eng.set_length(u, 47)
    q = np.ones((1, 8, D), np.float32)
    qr = c.rope(q, [47])
    out = torch.empty((1, 8 * D), device=DEV)
    c.eng.decode_attn(0, [u], dev(q), out)
    want, big = attention(qr, c.k[u][0].values[:48], c.v[u][0].values[:48], 47)
    err = np.abs(out.cpu().numpy().reshape(8, D) - want[0]).max()
    assert err <= attention_tolerance(big, 48, np.abs(c.v[u][0].values[:48]).max())


def test_rows_past_the_end_do_not_matter(cache8):
    """A page that held NaN, infinities and huge rows of another request."""
    rng = np.random.default_rng(41)
    c = cache8(G=8, n_pages=8)
    s = c.slot()
    bad = np.full((128, 8, D), np.nan, np.float32)
    bad[::2] = 3e38
    c.prefill(s, bad, bad)
    c.eng.release(s)
    slots = [c.slot() for _ in range(3)]
    for x, n in zip(slots, (3, 17, 20)):
        c.prefill(x, rows(rng, n, 8), rows(rng, n, 8))
    q, k, v = rng.standard_normal((3, 32, D)).astype(np.float32), rows(rng, 3, 8), rows(rng, 3, 8)
    out = torch.empty((3, 32 * D), device=DEV)
    c.eng.decode_step(0, slots, dev(q), dev(k), dev(v), out)
    for i, x in enumerate(slots):
        c.model_write(x, k[i:i + 1], v[i:i + 1])
    c.check_attention(slots, q, out)
    # a NaN row of its own poisons that slot's KV head and nothing else
    k[1, 3, 7] = np.nan
    c.eng.decode_step(0, slots, dev(q), dev(k), dev(v), out)
    o = out.view(3, 32, D).cpu().numpy()
    assert np.isnan(o[1, 12:16]).all() and np.isfinite(np.delete(o[1], range(12, 16), 0)).all()
    assert np.isfinite(o[[0, 2]]).all()


def test_shared_pages_are_copied_with_their_exponents(cache8):
    """fork in the middle of a page, then both sides append rows that outgrow it."""
    rng = np.random.default_rng(51)
    c = cache8(G=8, n_layers=3)
    s = c.slot()
    for layer in range(3):
        c.prefill(s, rows(rng, 37, 8), rows(rng, 37, 8), layer, advance=False)
    c.eng.advance([s], 37)
    t = c.eng.fork(s, 35)
    c.k[t], c.v[t] = [m.fork(35) for m in c.k[s]], [m.fork(35) for m in c.v[s]]
    for step in range(3):
        for layer in range(3):
            q, k, v = rng.standard_normal((2, 32, D)).astype(np.float32), rows(rng, 2, 8) * 3, rows(rng, 2, 8) * 9
            out = torch.empty((2, 32 * D), device=DEV)
            c.eng.decode_step(layer, [s, t], dev(q), dev(k), dev(v), out)
            for i, x in enumerate((s, t)):
                c.model_write(x, k[i:i + 1], v[i:i + 1], layer)
            c.check_attention([s, t], q, out, layer)
        c.eng.advance([s, t], 1)
    for layer in range(3):
        c.check(s, layer=layer)
        c.check(t, layer=layer)
    assert c.eng.stats()["cow_copies"] >= 1


def excess(got, want, bound):
    """By how much the worst element passes its bound."""
    return float((np.abs(got - want) - bound).max())


DTYPES = [("f32", torch.float32, 2.0 ** -24), ("f16", torch.float16, 2.0 ** -11), ("bf16", torch.bfloat16, 2.0 ** -8)]


@pytest.mark.parametrize("name,dt,half", DTYPES)
@pytest.mark.parametrize("cache", ["e4m3", "f16"])
@pytest.mark.parametrize("packed,norm", [(True, True), (False, False), (True, False), (False, True)])
def test_qkv_write(hkv_lib, oracle, rope_tables, name, dt, half, cache, packed, norm):
    """Norm and rotation of ragged rows of several slots, against float64.

    An F32 head is off by at most 40 * 2^-24 times (|a c| + |b s|) of its pair: the sum of
    squares (8 roundings in a tree), the root and the quotient (4), the products with the
    weight and the rotation (6); q_out adds half a step of its type (an F16 below 2^-14 has
    steps of 2^-24, so 2^-25 there; the other types have no such values here).  A cached value is within
    half an E4M3 step of that row (2^-4 of it, or 2^(e-10)), or half an F16 step."""
    import hkv
    G, H = 4, 16
    rng = np.random.default_rng(61)
    cos, sin = rope_tables
    eng = hkv.Engine(n_layers=2, n_head=H, n_head_kv=G, n_pages=64, max_slots=8, context_length=512, device=0,
                     shuffle_seed=3, cache=cache)
    slots = [eng.acquire() for _ in range(4)]
    old, new = [0, 13, 32, 7], [19, 1, 0, 40]
    for s, n in zip(slots, old):
        if n:
            z = torch.zeros((n, G, D), device=DEV)
            eng.rope_append_range(1, s, n, z, z)
            eng.advance([s], n)
    T = sum(new)
    if packed:
        x = torch.from_numpy(rng.standard_normal((T, (H + 2 * G) * D + 16)).astype(np.float32) * 2).to(DEV, dt)
        q, k, v = x[:, :H * D], x[:, H * D:(H + G) * D], x[:, (H + G) * D:(H + 2 * G) * D]
        strides = dict(q_stride=x.stride(0), k_stride=x.stride(0), v_stride=x.stride(0))
    else:
        q, k, v = (torch.from_numpy(rng.standard_normal((T, n * D)).astype(np.float32) * 2).to(DEV, dt) for n in (H, G, G))
        strides = {}
    qn, kn = dev(rng.random(D) + 0.5), dev(rng.random(D) + 0.5)
    eps = 1e-6
    q64, k64, v64 = (t.double().cpu().numpy().reshape(T, -1, D) for t in (q, k, v))
    if not packed:  # in place
        q_out = q
    else:
        q_out = torch.full((T + 1, H * D), 7.0, dtype=dt, device=DEV)
    eng.qkv_write(1, slots, new, q, k, v, q_norm=qn if norm else None, k_norm=kn if norm else None, eps=eps,
                  q_out=q_out, dtype=getattr(hkv, name.upper()), **strides)
    ko, vo = torch.empty((2, T, G, D), device=DEV).unbind(0)
    eng.cache_read(1, slots, old, new, ko, vo, dtype=hkv.F32)
    eng.sync_check()
    pos = np.concatenate([np.arange(p, p + n) for p, n in zip(old, new)])

    def want(x, w):
        if norm:
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.double().cpu().numpy()
        a, b = x[..., :64], x[..., 64:]
        c, s = cos[pos][:, None].astype(np.float64), sin[pos][:, None].astype(np.float64)
        y = np.concatenate([a * c - b * s, a * s + b * c], -1)
        m = np.concatenate([np.abs(a * c) + np.abs(b * s), np.abs(a * s) + np.abs(b * c)], -1)
        return y, 40 * 2.0 ** -24 * m

    floor = 2.0 ** -25 if name == "f16" else 0.0
    y, tol = want(q64, qn)
    got = q_out[:T].double().cpu().numpy().reshape(T, H, D)
    assert excess(got, y, tol + half * (np.abs(y) + tol) + floor) <= 0
    if packed:
        assert (q_out[T:].float() == 7.0).all()  # rows behind the last, as they were
    y, tol = want(k64, kn)
    ko, vo = ko.double().cpu().numpy(), vo.double().cpu().numpy()
    for got, x, t in ((ko, y, tol), (vo, v64, np.zeros_like(v64))):
        if cache == "f16":
            assert excess(got, x, t + 2.0 ** -11 * (np.abs(x) + t) + 2.0 ** -25) <= 0
            continue
        for e, n in enumerate(new):
            r = slice(sum(new[:e]), sum(new[:e + 1]))
            for g in range(G):
                for p in np.unique(pos[r] // PAGE):
                    rr = np.arange(r.start, r.stop)[pos[r] // PAGE == p]
                    step = 2.0 ** np.ceil(np.log2(np.abs(got[rr, g]).max() / 256))
                    bound = t[rr, g] + 2.0 ** -4 * (np.abs(x[rr, g]) + t[rr, g]) + step * 2.0 ** -10
                    assert excess(got[rr, g], x[rr, g], bound) <= 0
    # the rows of the other layer and of the slot without rows stay as they were
    z = torch.full((32, G, D), 3.0, device=DEV)
    z2 = z.clone()
    eng.cache_read(1, [slots[2]], [0], [32], z, z2, dtype=hkv.F32)
    assert (z == 0).all() and (z2 == 0).all()
    eng.close()


def test_qkv_write_equals_the_appends(cache8):
    """The same rows through hkv_qkv_write and through the append calls: the same bits."""
    rng = np.random.default_rng(71)
    import hkv
    a, b = cache8(G=8), cache8(G=8)
    sa, sb = [a.slot() for _ in range(3)], [b.slot() for _ in range(3)]
    for new in ([40, 3, 17], [1, 1, 1], [2, 0, 30]):
        k, v = rows(rng, sum(new), 8), rows(rng, sum(new), 8)
        a.eng.qkv_write(0, sa, new, None, dev(k), dev(v))
        at = 0
        for i, n in enumerate(new):
            if n:
                b.eng.rope_append_range(0, sb[i], n, dev(k[at:at + n]), dev(v[at:at + n]))
                a.eng.advance([sa[i]], n)
                b.eng.advance([sb[i]], n)
            at += n
    for x, y in zip(sa, sb):
        n = a.eng.length(x)
        assert n == b.eng.length(y)
        for p, q in zip(a.read(x, 0, n), b.read(y, 0, n)):
            assert np.array_equal(p, q)


def test_qkv_write_of_rotated_rows(cache8):
    """`rotated`: the rows go in as they are, and q comes out as it went in."""
    rng = np.random.default_rng(75)
    import hkv
    c = cache8(G=2)
    s = c.slot()
    k, v = rows(rng, 37, 2), rows(rng, 37, 2)
    q = rng.standard_normal((37, 8 * D)).astype(np.float32)
    out = torch.empty((37, 8 * D), device=DEV)
    c.eng.qkv_write(0, [s], [37], dev(q), dev(k), dev(v), q_out=out, rotated=True)
    c.model_write(s, k, v, roped=True)
    c.eng.advance([s], 37)
    c.check(s)
    assert np.array_equal(out.cpu().numpy(), q)
    with pytest.raises(hkv.HkvError, match="F16 caches"):  # what an 8-bit engine does not do
        c.eng.split_export(2, 0)


def test_calls_on_other_streams_and_engines(cache8):
    """Two engines on two streams in turn; the descriptor of one call outlives the next."""
    rng = np.random.default_rng(81)
    c = [cache8(G=8), cache8(G=8)]
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    slots = [[x.slot() for _ in range(3)] for x in c]
    for rep in range(6):
        keep = []
        for i in (0, 1):
            new = [int(n) for n in rng.integers(1, 40, 3)]
            k, v = rows(rng, sum(new), 8), rows(rng, sum(new), 8)
            dk, dv = dev(k), dev(v)
            torch.cuda.synchronize()
            c[i].eng.qkv_write(0, slots[i], new, None, dk, dv, stream=st[i].cuda_stream)
            at = 0
            for s, n in zip(slots[i], new):
                c[i].model_write(s, k[at:at + n], v[at:at + n])
                at += n
            for s, n in zip(slots[i], new):
                c[i].eng.advance([s], n)
            keep += [dk, dv]
        for x in st:
            x.synchronize()
    for i in (0, 1):
        for s in slots[i]:
            c[i].check(s)


def test_capture_is_refused(cache8):
    import hkv
    c = cache8(G=8)
    s = c.slot()
    z = torch.zeros((4, 8, D), device=DEV)
    c.prefill(s, np.zeros((4, 8, D), np.float32), np.zeros((4, 8, D), np.float32))
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        g.capture_begin()
        try:
            for call in (lambda: c.eng.qkv_write(0, [s], [4], None, z, z, stream=side.cuda_stream),
                         lambda: c.eng.cache_read(0, [s], [0], [4], z, z, dtype=hkv.F32, stream=side.cuda_stream)):
                with pytest.raises(hkv.HkvError, match="captured") as ei:
                    call()
                assert ei.value.status == hkv.HKV_ERR_INVALID
        finally:
            g.capture_end()
    c.check(s)


def test_range_append_in_a_capture_is_refused(cache8):
    import hkv
    c = cache8(G=1)
    s = c.slot()
    z = torch.zeros((4, 1, D), device=DEV)
    c.prefill(s, np.ones((4, 1, D), np.float32), np.ones((4, 1, D), np.float32))
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        g.capture_begin()
        try:
            with pytest.raises(hkv.HkvError, match="captured"):
                c.eng.rope_append_range(0, s, 4, z, z, stream=side.cuda_stream)
        finally:
            g.capture_end()
    c.check(s)


def test_backbone_runs_on_an_8_bit_cache(hkv_lib):
    """hkv_backbone_decode on an E4M3 engine: the fused step equals the calls it is made of."""
    import hkv
    from test_gpu_backbone import EPS, backbone_weights
    L, V = 2, 512
    w, _ = backbone_weights(hkv, L, V)
    engs = [hkv.Engine(n_layers=L, n_pages=64, max_slots=4, device=0, shuffle_seed=2, cache="e4m3") for _ in range(2)]
    bb = hkv.Backbone(engs[0], w, text_vocab=V, max_batch=2, rms_eps=EPS)
    slots = [[e.acquire(), e.acquire()] for e in engs]
    hid = torch.as_tensor(hkv.DeviceArray(bb.hidden_ptr, (2, 2560)), device=DEV)
    q, k, v, attn, g = (torch.empty((2, n), device=DEV) for n in (4096, 1024, 1024, 4096, 9728))
    for step in range(20):
        bb.embed_text([step + 1, 2 * step + 3])
        torch.cuda.synchronize()
        h = hid.clone()
        bb.decode(slots[0], want_logits=False)
        for l in range(L):
            p = f"blk.{l}."
            hkv.q4k_qkv(w[p + "attn_q"], w[p + "attn_k"], w[p + "attn_v"], 2560, h, w[p + "attn_q_norm"],
                        w[p + "attn_k_norm"], q, k, v, n=2, norm=w[p + "attn_norm"], eps=EPS, tensor_cores=True)
            engs[1].decode_step(l, slots[1], q, k, v, attn)
            hkv.q4k_gemv(w[p + "attn_output"], 2560, 4096, attn, h, n=2, residual=h, tensor_cores=True)
            hkv.q4k_gemv(w[p + "ffn_gate"], 9728, 2560, h, g, n=2, norm=w[p + "ffn_norm"], eps=EPS,
                         w_up=w[p + "ffn_up"], tensor_cores=True)
            hkv.q4k_gemv(w[p + "ffn_down"], 2560, 9728, g, h, n=2, residual=h, tensor_cores=True)
        engs[1].advance(slots[1], 1)
        torch.cuda.synchronize()
        assert torch.equal(h, hid)
    bb.sync_check()
    bb.close()
    for e in engs:
        e.sync_check()
        e.close()
