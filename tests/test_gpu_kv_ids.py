"""GPU tests of page ids outside the paged 8-bit cache: a plan does not take
them, a release does not put them on the free list, and either changes nothing."""
import numpy as np
import pytest

from tensai_b200 import KVCache, _lib
from test_gpu_kv import cu, i64, np_

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
PAGES = 4100


@pytest.fixture(scope="module", autouse=True)
def device():
    torch.cuda.init()
    _lib.check(_lib.load().tq_set_device(0))


@pytest.mark.parametrize("bad", [-1, PAGES, 2**31 - 1, -2**31])
@pytest.mark.parametrize("at", [0, 1, 1500, 3999])  # of the ids that the call takes
def test_a_plan_takes_no_page_outside_the_cache(bad, at):
    with KVCache(1, 1, 8, 16, PAGES) as cache:
        free = np.arange(PAGES)[::-1][:4050].copy()
        free[len(free) - 1 - at] = bad
        cached, added = np.array([5, 0, 16, 7]), np.array([1, 16 * 2000, 16 * 2000, 0])
        table = np.full((4, 2100), -1)
        table[0, 0], table[2, 0], table[3, 0] = 4096, 4097, 4098
        c, a, t, f, k = cu(cached), cu(added), cu(table), cu(free), cu([len(free)])
        s, ln, sl = cu([9] * 5), cu([9] * 4), i64([9] * (int(added.sum()) + 3))
        cache.plan(c, a, t, f, k, s, ln, sl)
        assert cache.status() == _lib.TQ_KV_STATUS_PAGE
        assert np.all(np_(s) == 0) and np.array_equal(np_(ln), cached) and np.all(np_(sl) == -1)
        assert np.array_equal(np_(t), table) and int(k) == len(free) and np.array_equal(np_(f), free)
        free[len(free) - 1 - at] = 4099  # put right, the same call does its work
        cache.plan(c, a, t, cu(free), k, s, ln, sl)
        assert cache.status() == 0 and int(k) == len(free) - 4000 and np.array_equal(np_(ln), cached + added)


def test_an_id_below_those_taken_is_not_looked_at():
    with KVCache(1, 1, 8, 16, 8) as cache:
        t, k = cu([[-1, -1]]), cu([3])
        cache.plan(cu([0]), cu([20]), t, cu([-1, 2, 3]), k, cu([0, 0]), cu([0]), i64([0] * 20))
        cache.check()
        assert np_(t).tolist() == [[3, 2]] and int(k) == 1


def test_held_positions_outside_the_cache_cost_their_own_tokens_alone():
    with KVCache(1, 1, 8, 16, 8) as cache:
        t, k, sl = cu([[9, -1], [1, -1]]), cu([3]), i64([7] * 6)
        cache.plan(cu([14, 3]), cu([4, 1]), t, cu([2, 3, 4]), k, cu([0] * 3), cu([0, 0]), sl)
        assert cache.status() == _lib.TQ_KV_STATUS_PAGE
        assert np_(sl).tolist() == [-1, -1, 64, 65, 19, 7] and int(k) == 2


@pytest.mark.parametrize("bad", [-1, PAGES, 2**31 - 1, -2**31])
@pytest.mark.parametrize("at", [0, 1, 2999])
def test_a_release_frees_no_page_outside_the_cache(bad, at):
    with KVCache(1, 1, 8, 16, PAGES) as cache:
        rows = np.arange(4000).reshape(2, 2000)
        rows = np.concatenate([rows, [[4000] + [-1] * 1999]])
        lens0, done = [16 * 1000, 16 * 2000 - 3, 1], [1, 1, 0]
        broken = rows.copy()
        i, b = (0, at) if at < 1000 else (1, at - 1000)
        broken[i, b] = bad
        lens, f, k = cu(lens0), cu([7] * 3100), cu([50])
        cache.release(cu(done), lens, cu(broken), f, k)
        assert cache.status() == _lib.TQ_KV_STATUS_PAGE
        assert list(np_(lens)) == lens0 and int(k) == 50 and bool((f == 7).all())
        cache.release(cu(done), lens, cu(rows), f, k)  # put right
        cache.check()
        assert list(np_(lens)) == [0, 0, 1] and int(k) == 3050
        assert np.array_equal(np_(f)[50:3050], np.concatenate([rows[0, :1000], rows[1]])) and bool((f[:50] == 7).all())
