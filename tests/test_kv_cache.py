"""CPU tests of the paged 8-bit cache: what its entry points refuse before any
device work, and the 64-bit restatement that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest

import kvref
from tensai_b200 import _lib


@pytest.fixture(scope="module")
def L():
    return _lib.load()


@pytest.mark.parametrize("cfg,msg", [
    ((0, 1, 64, 64, 1), "needs layers"),
    ((1, 0, 64, 64, 1), "needs layers"),
    ((1, 1, 64, 64, 0), "needs layers"),
    ((1, 65536, 64, 64, 1), "needs layers"),
    ((1, 1, 0, 64, 1), "head size"),
    ((1, 1, 12, 64, 1), "head size"),
    ((1, 1, 264, 64, 1), "head size"),
    ((1, 1, 64, 8, 1), "pages hold"),
    ((1, 1, 64, 48, 1), "pages hold"),
    ((1, 1, 64, 256, 1), "pages hold"),
])
def test_create_refuses_bad_shapes(L, cfg, msg):
    h = ctypes.c_uint64(7)
    assert L.tq_kv_create(ctypes.byref(_lib.KvConfig(*cfg)), ctypes.byref(h)) == _lib.TQ_ERR_ARG
    assert msg in L.tq_last_error().decode() and h.value == 7


def test_create_refuses_null_and_oversize(L):
    h = ctypes.c_uint64()
    assert L.tq_kv_create(None, ctypes.byref(h)) == _lib.TQ_ERR_ARG
    c = _lib.KvConfig(1, 65535, 256, 128, 2**31 - 1)
    assert L.tq_kv_create(ctypes.byref(c), ctypes.byref(h)) == _lib.TQ_ERR_UNSUPPORTED
    assert "too large" in L.tq_last_error().decode()


def test_unknown_cache_is_an_error(L):
    bits, size, dev = ctypes.c_uint(5), ctypes.c_size_t(5), ctypes.c_int()
    assert L.tq_kv_free(999) == _lib.TQ_OK  # as every free: a no-op
    for rc in (L.tq_kv_status(999, ctypes.byref(bits)), L.tq_kv_info(999, None, ctypes.byref(dev)),
               L.tq_kv_attention_workspace(999, ctypes.byref(size)),
               L.tq_kv_plan_dev(999, ctypes.byref(_lib.KvPlanArgs()), None),
               L.tq_kv_release_dev(999, ctypes.byref(_lib.KvReleaseArgs()), None),
               L.tq_kv_store_dev(999, 0, None, None, 0, 0, 0, None, 0, None),
               L.tq_kv_attention_dev(999, 0, ctypes.byref(_lib.KvAttentionArgs()), None),
               L.tq_kv_load_dev(999, 0, None, 0, None, None, None, None, None),
               L.tq_kv_save_dev(999, 0, None, 0, None, None, None, None, None),
               L.tq_kv_read_dev(999, 0, None, 0, None, None, None)):
        assert rc == _lib.TQ_ERR_HANDLE
        assert "invalid or freed cache handle" in L.tq_last_error().decode()
    assert bits.value == 0 and size.value == 0
    assert L.tq_kv_status(1, None) == _lib.TQ_ERR_ARG


def test_restated_store_holds_its_definition():
    """Codes within half a step of the stored values, scales the largest / 127,
    earlier codes rounded again when the scale grows."""
    rng = np.random.default_rng(1)
    ref = kvref.Ref(2, 16, 16, 3)
    x = rng.standard_normal((10, 2, 16))
    ref.store(x, 2 * x, np.arange(10) + 16)
    v = ref.values(0, np.array([1]))[0, :10]
    step = ref.scale[0][1].astype(np.float64)[None, :, None]
    assert np.all(np.abs(v - x) <= step * 0.5000001)
    assert np.allclose(ref.scale[0][1], np.abs(x).max((0, 2)) / 127, rtol=2**-23)
    before = ref.scale[0][1].copy()
    ref.store(100 * x[:1], x[:1], np.array([26]))
    assert np.all(ref.scale[0][1] > before) and np.array_equal(ref.scale[1][1], 2 * before)
    again = ref.values(0, np.array([1]))[0, :10]
    assert np.all(np.abs(again - v) <= ref.scale[0][1].astype(np.float64)[None, :, None] * 0.5000001)


def test_restated_attention_of_one_position_is_its_value():
    ref = kvref.Ref(1, 16, 16, 1)
    x = np.random.default_rng(2).standard_normal((1, 1, 16))
    ref.store(x, x, np.array([0]))
    out, mag, _, _ = ref.attention(x, [0, 1], [1], np.zeros((1, 1), int), 0.25)
    assert np.array_equal(out[0, 0], ref.values(1, np.array([0]))[0, 0, 0]) and np.array_equal(mag, np.abs(out))


def test_packed_arguments_are_the_structs_of_the_header():
    """kvcache.py packs its arguments; the ctypes structs state the header's layout."""
    from tensai_b200 import kvcache as K
    a = K._PLAN(1, 2, 3, 4, 5, *range(6, 15))
    s = _lib.KvPlanArgs(1, 2, 3, 4, 5, *range(6, 15))
    assert a == bytes(s)
    assert K._RELEASE(*range(1, 11)) == bytes(_lib.KvReleaseArgs(*range(1, 11)))
    v = (1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 0.5, 15, 16)
    assert K._ATTENTION(*v) == bytes(_lib.KvAttentionArgs(*v))
