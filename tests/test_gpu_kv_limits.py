"""GPU tests of what the paged 8-bit cache refuses before any launch: sizes whose
indexes would not stay ints in the kernels. The pointers are small arrays; no
call here reaches the device."""
import ctypes

import pytest

from tensai_b200 import KVCache, _lib
from test_gpu_kv import cu, i64

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
MOST = 2**31 - 1 - 65536


@pytest.fixture(scope="module", autouse=True)
def device():
    torch.cuda.init()
    _lib.check(_lib.load().tq_set_device(0))


def refused(rc, text):
    assert rc == _lib.TQ_ERR_UNSUPPORTED and text in _lib.load().tq_last_error().decode()


@pytest.mark.parametrize("page", [16, 128])
def test_sizes_next_to_two_to_the_31_are_refused(page):
    L = _lib.load()
    x, i = torch.zeros(64, device="cuda"), cu([0] * 8)
    j, s = [i[k:].data_ptr() for k in range(8)], i64([0]).data_ptr()
    cols = MOST // page + 1
    with KVCache(1, 1, 8, page, 1) as cache:
        def plan(cols=1, free=1, slots=1):
            return L.tq_kv_plan_dev(cache._h, ctypes.byref(_lib.KvPlanArgs(
                1, cols, cols, free, slots, j[0], j[1], j[2], j[3], j[4], j[5], j[7], s, j[4])), None)

        def release(cols=1, free=1):
            return L.tq_kv_release_dev(cache._h, ctypes.byref(_lib.KvReleaseArgs(
                1, cols, cols, free, j[0], j[1], j[2], j[3], j[4], j[4])), None)

        def attention(cols=1, tokens=1, heads=1):
            return L.tq_kv_attention_dev(cache._h, 0, ctypes.byref(_lib.KvAttentionArgs(
                x.data_ptr(), x.data_ptr(), 0, heads, tokens, 1, 2**40, 2**40, j[0], j[2], j[3], cols, cols, 1.0,
                x.data_ptr(), 0)), None)

        for call in (plan, release, attention):
            refused(call(cols=cols), "too long")
            refused(call(cols=2**31 - 1), "too long")
        refused(plan(slots=MOST + 1), "slots in one call")
        refused(plan(free=MOST + 1), "free pages in one call")
        refused(release(free=2**31 - 1), "free pages in one call")
        refused(attention(tokens=MOST + 1), "rows")
        refused(attention(tokens=2**20, heads=2**11), "rows")
        refused(L.tq_kv_store_dev(cache._h, 0, x.data_ptr(), x.data_ptr(), 0, 8, 8, s, MOST + 1, None), "tokens in one call")
        assert cache.status() == 0
