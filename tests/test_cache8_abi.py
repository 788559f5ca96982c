"""The 8-bit cache's entry points on a host-only engine (CPU): creation, the
slot bookkeeping, and every refusal, each before a GPU is asked for."""
from __future__ import annotations

import numpy as np
import pytest


@pytest.fixture
def eng(hkv_lib):
    import hkv
    e = hkv.Engine(n_layers=2, n_pages=64, max_slots=8, context_length=512, device=-1, lib=hkv_lib,
                   cache="e4m3")
    yield e
    e.close()


def test_create_with_a_cache_type(hkv_lib, eng):
    import hkv
    assert eng.cache == "e4m3"
    # codes of K and V and 32 bytes of exponents per (page, layer, KV head)
    assert eng.stats()["page_bytes"] == 2 * 8 * (2 * 16 * 128 + 32)
    f16 = hkv.Engine(n_layers=2, n_pages=4, max_slots=1, device=-1, lib=hkv_lib)
    assert f16.cache == "f16" and f16.stats()["page_bytes"] == 2 * 8 * 2 * 16 * 128 * 2
    f16.close()
    with pytest.raises(ValueError):
        hkv.Engine(n_layers=1, device=-1, lib=hkv_lib, cache="int4")
    h = hkv.ctypes.c_void_p()
    cfg = hkv.Config()
    assert hkv_lib.hkv_config_default(cfg) == 0
    cfg.device = -1
    for bad in (-1, 2, 99):
        assert hkv_lib.hkv_engine_create_cache(cfg, bad, h) == hkv.HKV_ERR_INVALID and not h.value
    assert hkv_lib.hkv_engine_create_cache(None, 1, h) == hkv.HKV_ERR_INVALID
    assert hkv_lib.hkv_engine_create_cache(cfg, 1, None) == hkv.HKV_ERR_INVALID


def test_slots_work_as_on_an_f16_engine(eng):
    s = eng.acquire(40)
    assert eng.stats()["reserved"] == 3
    eng.release(s)
    assert eng.stats()["free_pages"] == 64


def refused(eng, status, call, *args, **kw):
    import hkv
    before = eng.stats()
    with pytest.raises(hkv.HkvError) as ei:
        call(*args, **kw)
    assert ei.value.status == status, str(ei.value)
    assert eng.stats() == before


def test_qkv_write_refusals(eng):
    import hkv
    s, t = eng.acquire(0), eng.acquire(0)
    inv = hkv.HKV_ERR_INVALID
    w = eng.qkv_write
    refused(eng, inv, w, 0, [], [], None, 16, 16)
    refused(eng, hkv.HKV_ERR_BAD_SLOT, w, 0, [7], [1], None, 16, 16)
    refused(eng, inv, w, 0, [s, t, s], [1, 1, 1], None, 16, 16)
    refused(eng, hkv.HKV_ERR_RANGE, w, 0, [s], [-1], None, 16, 16)
    refused(eng, hkv.HKV_ERR_RANGE, w, 0, [s], [513], None, 16, 16)
    refused(eng, inv, w, 0, [s], [1], None, None, 16)
    refused(eng, inv, w, 0, [s], [1], None, 16, None)
    refused(eng, inv, w, 0, [s], [1], None, 24, 16)                      # not 16-byte aligned
    refused(eng, inv, w, 0, [s], [1], 16, 16, 16)                        # q without q_out
    refused(eng, inv, w, 0, [s], [1], None, 16, 16, q_out=16)            # q_out without q
    refused(eng, inv, w, 0, [s], [1], None, 16, 16, q_norm=16)           # q_norm without q
    refused(eng, inv, w, 0, [s], [1], 16, 16, 16, q_out=16, q_norm=20)   # misaligned weights
    refused(eng, inv, w, 0, [s], [1], None, 16, 16, k_norm=16, eps=-1.0)
    refused(eng, inv, w, 0, [s], [1], None, 16, 16, k_norm=16, eps=float("nan"))
    refused(eng, inv, w, 0, [s], [1], None, 16, 16, dtype=3)
    refused(eng, inv, w, 0, [s], [1], None, 16, 16, k_stride=1020)       # shorter than the row
    refused(eng, inv, w, 0, [s], [1], None, 16, 16, v_stride=1026)       # not whole 16-byte steps
    refused(eng, inv, w, 0, [s], [1], None, 16, 16, v_stride=1028, dtype=hkv.BF16)
    refused(eng, inv, w, 0, [s], [1], 16, 16, 16, q_out=16, q_stride=8192)  # in place, other stride
    refused(eng, hkv.HKV_ERR_NO_DEVICE, w, 0, [s], [1], None, 16, 16)    # nothing else is wrong
    with pytest.raises(ValueError):
        w(0, [s], [1, 2], None, 16, 16)


def test_cache_read_refusals(eng):
    import hkv
    s = eng.acquire(0)
    inv = hkv.HKV_ERR_INVALID
    r = eng.cache_read
    refused(eng, inv, r, 0, [], [], [], 16, 16)
    refused(eng, hkv.HKV_ERR_BAD_SLOT, r, 0, [5], [0], [1], 16, 16)
    refused(eng, hkv.HKV_ERR_RANGE, r, 0, [s], [0], [1], 16, 16)   # no row mapped
    refused(eng, hkv.HKV_ERR_RANGE, r, 0, [s], [-1], [0], 16, 16)
    refused(eng, hkv.HKV_ERR_RANGE, r, 0, [s], [0], [-1], 16, 16)
    refused(eng, inv, r, 0, [s], [0], [0], None, 16)
    refused(eng, inv, r, 0, [s], [0], [0], 16, 24)
    refused(eng, inv, r, 0, [s], [0], [0], 16, 16, dtype=hkv.BF16)
    refused(eng, inv, r, 0, [s, s], [0, 0], [0, 0], 16, 16)
    refused(eng, hkv.HKV_ERR_NO_DEVICE, r, 0, [s], [0], [0], 16, 16)


def test_window_attn_refusals(eng):
    import hkv
    s = eng.acquire(0)
    inv = hkv.HKV_ERR_INVALID
    w = eng.window_attn
    refused(eng, inv, w, 0, [], [], 16, 16)
    refused(eng, hkv.HKV_ERR_BAD_SLOT, w, 0, [5], [1], 16, 16)
    refused(eng, inv, w, 0, [s, s], [0, 0], 16, 16)
    refused(eng, hkv.HKV_ERR_RANGE, w, 0, [s], [-2], 16, 16)
    refused(eng, hkv.HKV_ERR_RANGE, w, 0, [s], [1], 16, 16)        # no row written
    refused(eng, inv, w, 0, [s], [0], None, 16)
    refused(eng, inv, w, 0, [s], [0], 16, 8)
    refused(eng, inv, w, 0, [s], [0], 16, 16, dtype=7)
    refused(eng, inv, w, 0, [s], [0], 16, 16, q_stride=4095)
    refused(eng, inv, w, 0, [s], [0], 16, 16, out_stride=4098)
    refused(eng, hkv.HKV_ERR_NO_DEVICE, w, 0, [s], [0], 16, 16)


def test_the_model_rounds_as_e4m3_does():
    """The model's own rounding against torch's E4M3 type over the whole range."""
    torch = pytest.importorskip("torch")
    from cache8_model import block_exponent, round_e4m3
    x = np.concatenate([np.linspace(-448, 448, 40001), np.geomspace(1e-6, 448, 20001),
                        np.arange(0, 64) * 2.0 ** -10]).astype(np.float32)
    t = torch.from_numpy(x).to(torch.float8_e4m3fn).to(torch.float64).numpy()
    assert np.array_equal(round_e4m3(x), t)
    for amax, e in ((448.0, 0), (np.nextafter(448, 500), 1), (449.0, 1), (224.0, -1), (1.75, -8),
                    (1.76, -7), (0.0, -100), (1e-40, -100), (3.4e38, 120)):
        assert block_exponent([amax]) == e, amax


def test_window_in_place_needs_equal_strides(eng):
    import hkv
    s = eng.acquire(0)
    refused(eng, hkv.HKV_ERR_INVALID, eng.window_attn, 0, [s], [0], 16, 16, q_stride=8192)
    refused(eng, hkv.HKV_ERR_NO_DEVICE, eng.window_attn, 0, [s], [0], 16, 16, q_stride=8192, out_stride=8192)
