"""GPU tests of the attention over the paged 8-bit cache: what a row does not
see must not reach it, whatever its scales are, and what weighs nothing must
not cost the rest its bits."""
import numpy as np
import pytest

import kvref
import kvrows
from tensai_b200 import KVCache, _lib
from test_gpu_kv import DT, batch, cu, i64, np_, widen

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
KINDS = [("f32", 3), ("bf16", 3), ("f16", 12)]  # two pieces, two pieces, one piece for p
LEAST = {"f32": 2.0**-140, "bf16": 2.0**-134, "f16": 2.0**-25}  # half a step of the type's least value


@pytest.fixture(scope="module", autouse=True)
def device():
    torch.cuda.init()
    _lib.check(_lib.load().tq_set_device(0))


def load(cache, ref):
    cache.load(0, cu(np.arange(len(ref.scale[0]))), *(cu(c, torch.int8) for c in ref.codes),
               *(cu(s, torch.float32) for s in ref.scale))


def compare(cache, ref, q, starts, lens, table, dtype, rows=None, many=False, scale=None):
    """The call's rows against the restatement; NaN where it has NaN."""
    n_q, hd = q.shape[1:]
    one = dtype != "f32" and (many or n_q // ref.n_kv > 8)
    wide = widen(table, len(q), n_q, hd, ref.page) if many else table
    out = np_(cache.attention(0, q, cu(starts), cu(lens), cu(wide), scale=scale))
    want, tol = kvrows.attend(ref, np_(q), starts, lens, table, hd**-0.5 if scale is None else scale,
                              torch.finfo(DT[dtype]).eps, one, many)
    rows = slice(None) if rows is None else rows
    assert np.array_equal(np.isnan(out[rows]), np.isnan(want[rows]))
    err = np.abs(out - want)[rows]
    ok = (err <= tol[rows] + LEAST[dtype]) | np.isnan(want[rows])
    assert np.all(ok), (int((~ok).sum()), float(np.nanmax(err / (tol[rows] + LEAST[dtype]))))


@pytest.mark.parametrize("dtype,group", KINDS)
@pytest.mark.parametrize("sides", [(0,), (1,), (0, 1)])
def test_a_scale_that_is_not_a_number_stays_with_the_rows_that_see_it(dtype, group, sides):
    """Two new tokens on two pages, the later page's scales not a number."""
    rng = np.random.default_rng(31)
    lens, new, page = [17, 40, 33], [2, 3, 1], 16
    cache, ref, table = batch(rng, 2, 64, page, lens)
    with cache:
        for side in sides:
            ref.scale[side][table[0, 1], 1] = np.float32("nan")  # position 16 of sequence 0, head 1
            ref.scale[side][table[1, 2], 0] = np.float32("nan")  # positions 32.. of sequence 1: all its rows
        load(cache, ref)
        starts = np.concatenate([[0], np.cumsum(new)])
        q = torch.tensor(rng.standard_normal((6, 2 * group, 64)), device="cuda").to(DT[dtype])
        compare(cache, ref, q, starts, lens, table, dtype)
        cache.check()


@pytest.mark.parametrize("dtype,group", KINDS)
def test_a_stored_key_that_is_not_finite_spoils_later_rows_alone(dtype, group):
    """As a program does it: two tokens stored, the second the first of a fresh
    page, its key infinite; then both attend."""
    rng = np.random.default_rng(32)
    with KVCache(1, 1, 64, 16, 2) as cache:
        ref = kvref.Ref(1, 64, 16, 2)
        k, v = (torch.tensor(rng.standard_normal((17, 1, 64)), device="cuda").to(DT[dtype]) for _ in range(2))
        k[16, 0, 9] = float("inf")
        cache.store(0, k, v, i64(np.arange(17)))
        ref.store(np_(k), np_(v), np.arange(17))
        q = torch.tensor(rng.standard_normal((2, group, 64)), device="cuda").to(DT[dtype])
        out = cache.attention(0, q, cu([0, 2]), cu([17]), cu([[0, 1]]))
        assert bool(torch.isfinite(out[0]).all()) and bool(torch.isnan(out[1]).all())
        compare(cache, ref, q, np.array([0, 2]), [17], np.array([[0, 1]]), dtype)


@pytest.mark.parametrize("dtype,group", KINDS)
@pytest.mark.parametrize("far", [2.0**30, 2.0**60])
def test_large_values_behind_a_row_cost_it_nothing(dtype, group, far):
    """The last token alone sees a page whose values are `far` times the others'."""
    rng = np.random.default_rng(33)
    lens, new, page = [33, 65], [3, 2], 16
    cache, ref, table = batch(rng, 1, 64, page, lens)
    with cache:
        ref.scale[1][table[0, 2]] *= np.float32(far)
        ref.scale[1][table[1, 4]] *= np.float32(far)
        load(cache, ref)
        q = torch.tensor(rng.standard_normal((5, group, 64)), device="cuda").to(DT[dtype])
        rows = [0, 1, 3] if dtype == "f16" else None  # the others are beyond float16
        compare(cache, ref, q, np.array([0, 3, 5]), lens, table, dtype, rows)
        cache.check()


@pytest.mark.parametrize("dtype,group", KINDS)
@pytest.mark.parametrize("many", [False, True])
def test_large_values_of_no_weight_cost_nothing(dtype, group, many):
    """A page that every row sees, of values 2^45 times the others', whose keys
    point away from the queries: scores about 300 below the others'."""
    rng = np.random.default_rng(34)
    new, page = (60 if many else 2), 16
    lens = [100]
    cache, ref, table = batch(rng, 1, 64, page, lens)
    with cache:
        u = rng.choice([-1.0, 1.0], 64)
        ref.codes[0][table[0, 1], :, 0] = -127 * u
        ref.scale[0][table[0, 1]] = 300 / (127 * 8)  # times 64 dimensions, times 64^-0.5
        ref.scale[1][table[0, 1]] *= np.float32(2.0**45)
        load(cache, ref)
        q = torch.tensor(u + 0.1 * rng.standard_normal((new, group, 64)), device="cuda").to(DT[dtype])
        compare(cache, ref, q, np.array([0, new]), lens, table, dtype, many=many)
        cache.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("small", [2.0**-20, 2.0**-40, 2.0**-60])
def test_small_values_beside_pages_of_zeros(dtype, many, small):
    """Every other page holds zeros, the rest values of `small`: the outputs are
    as exact as if the zeros were not there."""
    rng = np.random.default_rng(35)
    lens, new = [300, 77], ([100, 60] if many else [2, 1])
    cache, ref, table = batch(rng, 2, 64, 16, lens)
    with cache:
        for i in range(2):
            ids = table[i][table[i] >= 0]
            ref.scale[1][ids[::2]] = 0
            ref.scale[1][ids[1::2]] = np.float32(small)
        load(cache, ref)
        starts = np.concatenate([[0], np.cumsum(new)])
        q = torch.tensor(rng.standard_normal((starts[-1], 6, 64)), device="cuda").to(DT[dtype])
        compare(cache, ref, q, starts, lens, table, dtype, many=many)
        cache.check()
