"""Slot lists of the Python binding on a host-only engine (CPU): whatever int() takes one by one is
a list of slots, as are empty lists, where the C call takes them."""
from __future__ import annotations

from array import array

import numpy as np
import pytest


class Pointer:
    def data_ptr(self):
        return np.int64(16)


@pytest.fixture
def eng(hkv_lib):
    import hkv
    e = hkv.Engine(n_layers=1, n_pages=16, max_slots=4, context_length=64, device=-1, lib=hkv_lib)
    yield e
    e.close()


def lists(s, t):
    torch = pytest.importorskip("torch")
    return [[s, t], (s, t), [float(s), float(t)], np.array([s, t]), np.array([s, t], np.float32), np.array([s, t], np.uint8),
            array("q", [s, t]), array("f", [s, t]), torch.tensor([s, t]), torch.tensor([float(s), float(t)]),
            [str(s), t], bytes([s, t]), bytearray([s, t]), {s: 0, t: 0}, [np.int64(s), np.float64(t)]]


def test_what_a_slot_list_may_be(eng):
    """Without a device, a call that found its slots live says so; an unknown one is refused before."""
    import hkv
    s, t = eng.acquire(16), eng.acquire(16)
    for slots in lists(s, t):
        eng.advance(slots, 0)
        for call in (lambda: eng.append(0, slots, 16, 16), lambda: eng.decode_attn(0, slots, 16, 16),
                     lambda: eng.qkv_write(0, slots, [1, 1], None, 16, 16),
                     lambda: eng.window_attn(0, slots, [0, 0], 16, 16)):
            with pytest.raises(hkv.HkvError) as e:
                call()
            assert e.value.status == hkv.HKV_ERR_NO_DEVICE, slots
    for wrong in ([s, 3], [s, -1], [2 ** 31, s], [s, 2 ** 32 + t]):
        with pytest.raises(hkv.HkvError) as e:
            eng.advance(wrong, 0)
        assert e.value.status == hkv.HKV_ERR_BAD_SLOT, wrong
    eng.advance([], 0)
    for bad in ([None], [s, "x"]):
        with pytest.raises((TypeError, ValueError)):
            eng.advance(bad, 0)
    with pytest.raises(hkv.HkvError) as e:  # a pointer that is a numpy integer
        eng.qkv_write(0, [s], [1], None, Pointer(), Pointer())
    assert e.value.status == hkv.HKV_ERR_NO_DEVICE
