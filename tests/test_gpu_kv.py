"""GPU tests of the paged 8-bit cache (tensai_b200.KVCache, through the C ABI)
against its 64-bit restatement (kvref.py): plans and slots equal, codes and
scales bit for bit, attention within a bound from the arithmetic of its parts,
over types, head sizes, groups, page sizes, ragged lengths, captured graphs."""
import numpy as np
import pytest

import kvref
from tensai_b200 import KVCache, TensaiError, _lib

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module", autouse=True)
def device():
    torch.cuda.init()
    _lib.check(_lib.load().tq_set_device(0))


def cu(x, dtype=torch.int32):
    return torch.tensor(np.asarray(x), dtype=dtype, device="cuda")


def i64(x):
    return cu(x, torch.int64)


def np_(t):
    return t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


# ---- plan ------------------------------------------------------------------------------

def plan_inputs(rng, n, page, most, new):
    cached = rng.integers(0, most + 1, n)
    added = np.where(rng.random(n) < 0.2, rng.integers(0, new + 1, n), 1)
    need = sum(kvref.pages(c, page) for c in cached)
    grow = sum(kvref.pages(c + a, page) - kvref.pages(c, page) for c, a in zip(cached, added))
    ids = rng.permutation(need + grow + 5)
    width = max([kvref.pages(c + a, page) for c, a in zip(cached, added)] + [1])
    table = np.full((n, width), -1)
    at = 0
    for i, c in enumerate(cached):
        m = kvref.pages(c, page)
        table[i, :m] = ids[at:at + m]
        at += m
    return cached, added, table, ids[at:], need + grow + 5


@pytest.mark.parametrize("n,page,most,new", [(0, 16, 1, 1), (1, 16, 0, 1), (1, 64, 100, 5000), (7, 32, 40, 3),
                                             (300, 128, 500, 64), (1500, 16, 300, 200), (16384, 64, 200, 2)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_matches_the_restatement(n, page, most, new, in_place):
    cached, added, table, free, n_pages = plan_inputs(np.random.default_rng(n + page), n, page, most, new)
    starts, lens, slots, want, left = kvref.plan(cached, added, table, free, page)
    with KVCache(1, 1, 8, page, n_pages) as cache:
        c, a, t = cu(cached), cu(added), cu(table).reshape(n, table.shape[1])
        f, count = cu(free), cu([len(free)])
        s, sl = torch.full((n + 1,), -7, dtype=torch.int32, device="cuda"), i64(np.full(len(slots) + 3, -9))
        ln, lf = (c, count) if in_place else (torch.empty_like(c), torch.empty_like(count))
        cache.plan(c, a, t, f, count, s, ln, sl, free_left=None if in_place else lf)
        cache.check()
        assert np.array_equal(np_(s), starts) and np.array_equal(np_(ln), lens)
        assert np.array_equal(np_(sl)[:len(slots)], slots) and np.all(np_(sl)[len(slots):] == -9)
        assert np.array_equal(np_(t), want) and int(lf) == len(left)
        assert np.array_equal(np_(f), free)


@pytest.mark.parametrize("break_it,bit", [("pool", _lib.TQ_KV_STATUS_POOL), ("table", _lib.TQ_KV_STATUS_TABLE),
                                          ("slots", _lib.TQ_KV_STATUS_SLOTS), ("cached", _lib.TQ_KV_STATUS_LENGTH),
                                          ("added", _lib.TQ_KV_STATUS_LENGTH), ("count", _lib.TQ_KV_STATUS_LENGTH)])
def test_a_plan_that_does_not_fit_changes_nothing(break_it, bit):
    cached, added, table = np.array([16, 3, 40]), np.array([1, 20, 0]), np.array([[4, -1], [5, -1], [6, 7]])
    page, free = 32, np.array([0, 1, 2, 3])
    if break_it == "table":
        added[2] = 25
    if break_it in ("cached", "added"):
        dict(cached=cached, added=added)[break_it][1] = -1
    count = dict(pool=0, count=5).get(break_it, 4)
    if break_it == "pool":
        added[1] = 30
    with KVCache(1, 1, 8, page, 8) as cache:
        c, a, t, f, k = cu(cached), cu(added), cu(table), cu(free), cu([count])
        s, ln, sl = cu([9] * 4), cu([9] * 3), i64([9] * (20 if break_it == "slots" else 60))
        cache.plan(c, a, t, f, k, s, ln, sl)
        with pytest.raises(TensaiError, match="tensai: cache"):
            cache.plan(c, a, t, f, k, s, ln, sl)
            cache.check()
        assert cache.status() == 0
        cache.plan(c, a, t, f, k, s, ln, sl)
        assert cache.status() == bit
        assert np.all(np_(s) == 0) and np.array_equal(np_(ln), cached) and np.all(np_(sl) == -1)
        assert np.array_equal(np_(t), table) and int(k) == count
        # what stands behind it in the stream does nothing
        x = torch.ones((len(sl), 1, 8), device="cuda")
        cache.store(0, x, x, sl)
        out = torch.full_like(x, 5)
        cache.attention(0, x, s, cu([1, 1, 1]), t, out=out)
        assert cache.status() == 0 and bool((out == 5).all())
        assert not any(bool(y.any()) for y in cache.read(0, cu(np.arange(8))))


def test_plans_and_releases_never_share_a_page():
    rng = np.random.default_rng(5)
    n, page, n_pages = 40, 16, 400
    with KVCache(1, 1, 8, page, n_pages) as cache:
        lens = cu(np.zeros(n))
        table, free, count = cu(np.full((n, 24), -1)), cu(rng.permutation(n_pages)), cu([n_pages])
        starts, slots = cu(np.zeros(n + 1)), i64(np.zeros(n * 30))
        for step in range(60):
            now = np_(lens)
            room = np.maximum(0, np.minimum(30, 24 * page - now))
            added = np.minimum(room, rng.integers(0, 31, n) * (rng.random(n) < 0.5))
            if sum(kvref.pages(v, page) for v in now + added) <= n_pages:
                cache.plan(lens, cu(added), table, free, count, starts, lens, slots)
                now = now + added
                assert np.array_equal(np_(lens), now)
            done = (rng.random(n) < 0.08).astype(np.int64)
            cache.release(cu(done), lens, table, free, count)
            now = np.where(done, 0, now)
            cache.check()
            t, k = np_(table), int(count)
            held = [int(t[i, b]) for i in range(n) for b in range(kvref.pages(now[i], page))]
            assert np.array_equal(np_(lens), now) and k == n_pages - len(held)
            assert sorted(held + list(np_(free)[:k])) == list(range(n_pages))


def test_release_refuses_on_the_device():
    with KVCache(1, 1, 8, 16, 8) as cache:
        lens, table, free, k = cu([20, 5]), cu([[1, 2], [3, 4]]), cu([0, 5, 6]), cu([2])
        cache.release(cu([1, 0]), lens, table, free, k)  # two pages into one free place
        assert cache.status() == _lib.TQ_KV_STATUS_POOL
        assert list(np_(lens)) == [20, 5] and int(k) == 2 and list(np_(free)) == [0, 5, 6]
        cache.release(cu([0, 1]), lens, table, free, k)
        assert cache.status() == 0 and list(np_(lens)) == [20, 0] and int(k) == 3 and list(np_(free)) == [0, 5, 3]
        cache.release(cu([1, 0]), cu([40, 0]), table, cu([0] * 9), cu([0]))
        assert cache.status() == _lib.TQ_KV_STATUS_TABLE


# ---- store -----------------------------------------------------------------------------

def codes_equal(cache, ref, ids, layer=0):
    k, v, ks, vs = cache.save(layer, cu(ids))
    for got, want in ((ks, ref.scale[0]), (vs, ref.scale[1])):
        assert np.array_equal(got.cpu().numpy(), want[ids], equal_nan=True)
    for got, want in ((k, ref.codes[0]), (v, ref.codes[1])):
        assert np.array_equal(got.cpu().numpy(), want[ids])


def random_pages(cache, ref, rng):
    """Every page holds something already, as recycled pages do."""
    for side in range(2):
        ref.codes[side][:] = rng.integers(-127, 128, ref.codes[side].shape)
        ref.scale[side][:] = rng.random(ref.scale[side].shape) * 0.02
    n = len(ref.scale[0])
    for layer in range(cache.n_layer):
        cache.load(layer, cu(np.arange(n)), *(cu(c, torch.int8) for c in ref.codes),
                   *(cu(s, torch.float32) for s in ref.scale))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_kv,hd,page,runs", [
    (1, 8, 16, [(0, 1)]), (2, 64, 16, [(5, 1), (15, 1), (0, 1)]), (3, 80, 32, [(7, 60), (0, 33)]),
    (4, 128, 64, [(63, 2), (1, 200)]), (2, 256, 128, [(100, 200), (0, 128)]), (12, 40, 64, [(16, 16), (17, 31)]),
    (2, 72, 128, [(3, 1200)])])
def test_store_bit_for_bit(dtype, n_kv, hd, page, runs):
    """runs: (tokens held, tokens added) per sequence; pages in random order."""
    rng = np.random.default_rng(hd * page + n_kv)
    need = [kvref.pages(c + a, page) for c, a in runs]
    n_pages = sum(need) + 2
    ids = rng.permutation(n_pages)
    slots, at = [], 0
    for (c, a), m in zip(runs, need):
        mine = ids[at:at + m]
        at += m
        slots += [int(mine[p // page]) * page + p % page for p in range(c, c + a)]
    T = len(slots)
    with KVCache(2, n_kv, hd, page, n_pages) as cache:
        ref = kvref.Ref(n_kv, hd, page, n_pages)
        random_pages(cache, ref, rng)
        k, v = (torch.tensor(rng.standard_normal((T, n_kv, hd)) * s, device="cuda").to(DT[dtype]) for s in (3, 0.1))
        cache.store(1, k, v, i64(slots))
        cache.check()
        untouched = kvref.Ref(n_kv, hd, page, n_pages)
        untouched.codes, untouched.scale = [c.copy() for c in ref.codes], [s.copy() for s in ref.scale]
        ref.store(np_(k), np_(v), slots)
        codes_equal(cache, ref, np.arange(n_pages), 1)
        codes_equal(cache, untouched, np.arange(n_pages), 0)


@pytest.mark.parametrize("dtype,n_kv,hd,page,T", [("f32", 12, 8, 32, 4000), ("bf16", 12, 16, 16, 2500), ("f32", 2, 256, 128, 700),
                                                  ("f16", 2, 256, 128, 130)])
def test_store_of_many_runs(dtype, n_kv, hd, page, T):
    """Runs of all lengths that begin anywhere in a page, skipped tokens between
    them: blocks that look for several runs, and blocks of 1,024 threads."""
    rng = np.random.default_rng(T)
    slots, at = [], 0
    while len(slots) < T:
        if rng.random() < 0.2:
            slots += [-1] * int(rng.integers(1, 4))
        off = int(rng.integers(0, page))
        run = int(rng.integers(1, 3)) if rng.random() < 0.5 else int(rng.integers(1, 3 * page))
        for p in range(off, off + run):
            slots.append((at + p // page) * page + p % page)
        at += (off + run - 1) // page + 1
    slots, n_pages = slots[:T], at
    with KVCache(1, n_kv, hd, page, n_pages) as cache:
        ref = kvref.Ref(n_kv, hd, page, n_pages)
        random_pages(cache, ref, rng)
        k, v = (torch.tensor(rng.standard_normal((T, n_kv, hd)) * s, device="cuda").to(DT[dtype]) for s in (3, 0.1))
        cache.store(0, k, v, i64(slots))
        cache.check()
        ref.store(np_(k), np_(v), slots)
        codes_equal(cache, ref, np.arange(n_pages))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_token_by_token_appends(dtype):
    """A page filled one token at a time, its scale growing on the way."""
    rng = np.random.default_rng(3)
    with KVCache(1, 2, 64, 32, 3) as cache:
        ref = kvref.Ref(2, 64, 32, 3)
        random_pages(cache, ref, rng)
        for t in range(70):
            x = torch.tensor(rng.standard_normal((2, 1, 2, 64)) * 1.05**t, device="cuda").to(DT[dtype])
            slot = [(2 - t // 32) * 32 + t % 32]
            cache.store(0, x[0], x[1], i64(slot))
            ref.store(np_(x[0]), np_(x[1]), slot)
            if t % 9 == 0 or t == 69:
                codes_equal(cache, ref, np.arange(3))


def test_ties_and_near_ties():
    """Quotients at and beside n + 1/2: ties to even, neighbours to their side."""
    s = np.float32(0.75)
    n = np.arange(-126, 126)
    halves = ((n + 0.5) * float(s)).astype(np.float32)  # exact: 0.75 has two bits
    x = np.concatenate([halves, np.nextafter(halves, np.float32(np.inf)), np.nextafter(halves, np.float32(-np.inf)),
                        [np.float32(127 * 0.75)] * 12])
    rng = np.random.default_rng(4)
    odd = np.float32(0.0123)  # a scale with all its bits: the nearest floats to the halves
    y = np.concatenate([np.float32((n + 0.5) * float(odd))] * 3 + [[np.float32(127 * float(odd))] * 12])
    z = np.concatenate([rng.permutation(y)])
    with KVCache(1, 1, 256, 16, 2) as cache:
        ref = kvref.Ref(1, 256, 16, 2)
        for arr in (x, z):
            t = torch.tensor(arr[:768].reshape(3, 1, 256), device="cuda")
            cache.store(0, t, -t, i64([0, 1, 2]))
            ref.store(np_(t), -np_(t), [0, 1, 2])
            codes_equal(cache, ref, [0])


@pytest.mark.parametrize("size", [0.0, 1e-45, 1e-40, 1e-37, 3e-31, 1e30, 3e38])
def test_extreme_magnitudes(size):
    rng = np.random.default_rng(6)
    x = torch.tensor((rng.standard_normal((5, 1, 32)).clip(-1, 1) * size).astype(np.float32), device="cuda")
    with KVCache(1, 1, 32, 16, 2) as cache:
        ref = kvref.Ref(1, 32, 16, 2)
        cache.store(0, x, x * 0.5, i64([16, 17, 18, 19, 20]))
        ref.store(np_(x), np_(x * 0.5), [16, 17, 18, 19, 20])
        codes_equal(cache, ref, [0, 1])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_value_that_is_not_finite_spoils_its_page_and_head_alone(bad):
    rng = np.random.default_rng(7)
    x = torch.tensor(rng.standard_normal((40, 2, 16)), device="cuda", dtype=torch.float32)
    x[20, 1, 3] = bad
    slots = np.arange(40)
    with KVCache(1, 2, 16, 16, 3) as cache:
        ref = kvref.Ref(2, 16, 16, 3)
        cache.store(0, x, x, i64(slots))
        ref.store(np_(x), np_(x), slots)
        codes_equal(cache, ref, [0, 1, 2])
        k, _ = cache.read(0, cu([0, 1, 2]))
        assert bool(torch.isnan(k[1, :, 1]).all()) and not bool(torch.isnan(k[[0, 2]]).any())
        assert not bool(torch.isnan(k[1, :, 0]).any())
        # an append keeps it, the page's first position clears it
        for slot in (40, 16):
            cache.store(0, x[:1], x[:1], i64([slot]))
            ref.store(np_(x[:1]), np_(x[:1]), [slot])
        codes_equal(cache, ref, [0, 1, 2])


def test_strided_unaligned_and_skipped_tokens():
    rng = np.random.default_rng(8)
    fused = torch.tensor(rng.standard_normal((9, 1 + 5 * 48)), device="cuda").to(torch.bfloat16)
    k, v = fused[:, 1:97].view(9, 2, 48), fused[:, 97:193].unflatten(1, (2, 48))
    slots = [3, -1, 4, 5, 64, 65, -5, 31, 95]
    with KVCache(1, 2, 48, 32, 3) as cache:
        ref = kvref.Ref(2, 48, 32, 3)
        random_pages(cache, ref, rng)
        slots[2:4] = [40, 41]
        cache.store(0, k, v, i64(slots[:7] + [-1, -1]))
        ref.store(np_(k), np_(v), slots[:7] + [-1, -1])
        cache.check()
        codes_equal(cache, ref, [0, 1, 2])


def test_bad_slots_are_skipped_and_reported():
    rng = np.random.default_rng(9)
    x = torch.tensor(rng.standard_normal((4, 1, 16)), device="cuda", dtype=torch.float32)
    with KVCache(1, 1, 16, 16, 3) as cache:
        ref = kvref.Ref(1, 16, 16, 3)
        cache.store(0, x, x, i64([0, 48, 2**40, 33]))
        assert cache.status() == _lib.TQ_KV_STATUS_PAGE
        ref.store(np_(x), np_(x), [0, -1, -1, 33])
        codes_equal(cache, ref, [0, 1, 2])
        cache.store(0, x, x, i64([20, 20, 18, 0]))  # the same slot again, then a smaller one: the first counts
        assert cache.status() == _lib.TQ_KV_STATUS_SLOTS
        ref.store(np_(x), np_(x), [20, -1, -1, 0])
        codes_equal(cache, ref, [0, 1, 2])
        cache.store(0, x[:0], x[:0], i64([]))
        cache.check()


def test_pages_in_and_out():
    rng = np.random.default_rng(10)
    with KVCache(2, 3, 40, 32, 6) as cache:
        ref = kvref.Ref(3, 40, 32, 6)
        random_pages(cache, ref, rng)
        codes_equal(cache, ref, [5, 0, 3])
        k, v = cache.read(1, cu([4, 4, 1]))
        for got, side in ((k, 0), (v, 1)):
            want = ref.codes[side][[4, 4, 1]].astype(np.float32) * ref.scale[side][[4, 4, 1]][:, None, :, None]
            assert np.array_equal(got.cpu().numpy(), want)
        low = torch.full((1, 32, 3, 40), -128, dtype=torch.int8, device="cuda")
        one = torch.ones((1, 3), device="cuda")
        cache.load(0, cu([2]), low, low, one, one)
        assert bool((cache.save(0, cu([2]))[0] == -127).all())
        cache.read(0, cu([6, -1]))
        assert cache.status() == _lib.TQ_KV_STATUS_PAGE


# ---- attention --------------------------------------------------------------------------

def batch(rng, n_kv, hd, page, lens, extra=3, wide=1.0):
    """A cache with random pages, and a table of random distinct pages for the lengths."""
    need = [kvref.pages(v, page) for v in lens]
    n_pages = sum(need) + extra
    ids = rng.permutation(n_pages)
    table = np.full((len(lens), max(need + [1]) + 1), -1)
    at = 0
    for i, m in enumerate(need):
        table[i, :m] = ids[at:at + m]
        at += m
    ref = kvref.Ref(n_kv, hd, page, n_pages)
    cache = KVCache(1, n_kv, hd, page, n_pages)
    random_pages(cache, ref, rng)
    if wide != 1.0:
        for side in range(2):
            ref.scale[side] *= wide ** rng.integers(-1, 2, ref.scale[side].shape).astype(np.float32)
        cache.load(0, cu(np.arange(n_pages)), *(cu(c, torch.int8) for c in ref.codes),
                   *(cu(s, torch.float32) for s in ref.scale))
    return cache, ref, table


def widen(table, tokens, n_q, hd, page):
    """The same table in rows so wide that many rows go to the tensor-memory
    kernel, whatever the lengths are."""
    hdp = 64 if hd <= 64 else 128
    cols = max(table.shape[1], int(512e6 / (tokens * n_q * hdp * page)) + 2)
    out = np.full((table.shape[0], cols), -1)
    out[:, :table.shape[1]] = table
    return out


def bound(ref_out, mag, qk, top_v, dtype, hd, group, longest, new, many=False):
    """What the arithmetic allows. Per position: the score's hd products (22 bits
    of q, float32 sums that the tensor cores may truncate: 2^-22 each) move p by
    twice their error; exp2 and the pieces of p 2^-21; 2^-12 where p is one
    float16 (16-bit queries, more than eight heads to a KV head or many rows);
    every addition over the positions 2^-22; then the output's own rounding.
    p times its value scale, over the largest value scale, is held in float16 at
    2^14 for p = 1, whose steps below 2^-14 are 2^-24: a rounding of at most
    2^-25 / 2^14 = 2^-39 of the largest value for each position, whatever p is
    (after division by the sum of p, which is at least 1). With many rows the
    unit is 2^10 for the largest p times its scale, or up to 2^4 below that:
    2^-25 / 2^10 = 2^-35."""
    one = dtype != "f32" and (group > 8 or many)
    rel = 2 * (hd + 16) * 2.0**-22 * qk + (longest + 64) * 2.0**-22 + 2.0**-21 + (2.0**-11 if one else 0)
    half = torch.finfo(DT[dtype]).eps / 2
    floor = longest * (2.0**-35 if many else 2.0**-39) * top_v
    return mag * rel[..., None] + floor[..., None] + np.abs(ref_out) * half * 1.0001 + 2.0**-24 * half


def run_attention(cache, ref, table, lens, new, dtype, n_q, rng, scale=None, q_scale=1.0, pad=2):
    starts = np.concatenate([[0], np.cumsum(new)])
    T, hd = int(starts[-1]), ref.hd
    q = torch.tensor(rng.standard_normal((T + pad, n_q, hd)) * q_scale, device="cuda").to(DT[dtype])
    want, mag, qk, top_v = ref.attention(np_(q), starts, lens, table, hd**-0.5 if scale is None else scale)
    group = n_q // ref.n_kv
    for many in (False, True):
        if many and (hd > 128 or max(new, default=0) * group <= 48):
            break
        out = torch.full_like(q, 7)
        rows = widen(table, T, n_q, hd, ref.page) if many else table
        cache.attention(0, q, cu(starts), cu(lens), cu(rows), out=out, scale=scale)
        got = np_(out)
        assert np.all(got[T:] == 7)
        tol = bound(want, mag, qk, top_v, dtype, hd, group, max(lens, default=0), new, many)
        err = np.abs(got - want)[:T]
        assert np.all(err <= tol[:T]), (many, float(np.max(err - tol[:T])), float(np.max(err)))
    return q, out


SHAPES = [  # n_kv, group, hd, page
    (1, 1, 64, 16), (2, 7, 128, 64), (4, 2, 128, 16), (1, 16, 64, 32), (2, 3, 80, 32), (1, 9, 128, 128),
    (3, 1, 256, 64), (1, 33, 96, 16), (2, 4, 8, 128), (1, 20, 256, 16)]
LENS = [1, 0, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 1000]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_kv,group,hd,page", SHAPES)
def test_decode_attention(dtype, n_kv, group, hd, page):
    rng = np.random.default_rng(hd + page + group)
    cache, ref, table = batch(rng, n_kv, hd, page, LENS)
    with cache:
        run_attention(cache, ref, table, LENS, [1] * len(LENS), dtype, n_kv * group, rng, q_scale=2.0)
        cache.check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n_kv,group,hd,page", SHAPES)
def test_attention_of_several_tokens(dtype, n_kv, group, hd, page):
    """Prompts, pieces of prompts, rows without tokens, and more queries than
    positions (whose first rows see nothing and are 0)."""
    rng = np.random.default_rng(7 * hd + page + group)
    lens = [1, 5, 40, 64, 100, 130, 3, 0, 300]
    new = [1, 5, 7, 64, 33, 130, 6, 2, 150]
    cache, ref, table = batch(rng, n_kv, hd, page, lens)
    with cache:
        _, out = run_attention(cache, ref, table, lens, new, dtype, n_kv * group, rng, q_scale=2.0)
        cache.check()
        starts = np.concatenate([[0], np.cumsum(new)])
        assert not bool(out[starts[6]:starts[6] + 3].any()) and not bool(out[starts[7]:starts[8]].any())


@pytest.mark.parametrize("dtype,n_kv,group,hd", [("f32", 1, 4, 128), ("bf16", 2, 7, 128), ("f16", 1, 1, 64),
                                                 ("bf16", 1, 12, 256)])
def test_long_contexts_split_over_the_gpu(dtype, n_kv, group, hd):
    rng = np.random.default_rng(11)
    lens = [30011, 1, 517]
    cache, ref, table = batch(rng, n_kv, hd, 64, lens)
    with cache:
        q, out = run_attention(cache, ref, table, lens, [1, 1, 1], dtype, n_kv * group, rng, q_scale=3.0)
        again = cache.attention(0, q, cu([0, 1, 2, 3]), cu(lens), cu(table))
        assert torch.equal(again[:3], out[:3])  # the same bits


@pytest.mark.parametrize("n", [513, 1500])
def test_many_sequences(n):
    rng = np.random.default_rng(n)
    lens = list(rng.integers(0, 90, n))
    cache, ref, table = batch(rng, 1, 16, 16, lens)
    with cache:
        run_attention(cache, ref, table, lens, list(rng.integers(0, 3, n)), "f32", 2, rng)
        cache.check()


@pytest.mark.parametrize("n", [40, 600, 1300])
def test_many_sequences_some_with_many_rows(n):
    rng = np.random.default_rng(n)
    lens = list(rng.integers(0, 90, n))
    new = list(rng.integers(0, 3, n))
    for i in range(3, n, 17):  # some as long as their sequence, or a row short of the other kernel's
        new[i] = min(int(lens[i]), [30, 24, 25, 90][i % 4])
    cache, ref, table = batch(rng, 1, 16, 16, lens)
    with cache:
        run_attention(cache, ref, table, lens, new, "bf16", 2, rng)
        cache.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("wide", [2.0**6, 2.0**-9])
def test_scales_far_apart(dtype, wide):
    """Neighbouring pages whose scales differ by up to 2^18."""
    rng = np.random.default_rng(12)
    lens = [200, 64, 333]
    cache, ref, table = batch(rng, 2, 64, 16, lens, wide=wide)
    for side in range(2):
        assert ref.scale[side].min() >= 0
    with cache:
        run_attention(cache, ref, table, lens, [1, 3, 40], dtype, 8, rng, q_scale=1.0)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_scale", [0.0, 1e-30, 1e-4, 300.0])
def test_query_magnitudes(dtype, q_scale):
    rng = np.random.default_rng(13)
    lens = [77, 5]
    cache, ref, table = batch(rng, 1, 64, 32, lens)
    with cache:
        run_attention(cache, ref, table, lens, [2, 1], dtype, 3, rng, scale=0.7 if q_scale else 0.0, q_scale=q_scale)


@pytest.mark.parametrize("dtype,group", [("f32", 3), ("bf16", 3), ("f16", 12)])
def test_a_negative_score_factor(dtype, group):
    rng = np.random.default_rng(27)
    lens, new = [90, 33, 260], [60, 1, 70]
    cache, ref, table = batch(rng, 2, 64, 32, lens)
    with cache:
        run_attention(cache, ref, table, lens, new, dtype, 2 * group, rng, scale=-0.2)
        cache.check()


def test_zero_scales_and_equal_scores():
    rng = np.random.default_rng(14)
    cache, ref, table = batch(rng, 1, 32, 16, [50])
    with cache:
        ref.scale[0][:] = 0  # values 0 whatever the codes are
        ref.scale[1][table[0, 1]] = 0
        cache.load(0, cu(np.arange(len(ref.scale[0]))), *(cu(c, torch.int8) for c in ref.codes),
                   *(cu(s, torch.float32) for s in ref.scale))
        run_attention(cache, ref, table, [50], [4], "f32", 2, rng)
        ref.scale[1][:] = 0  # all values zero
        cache.load(0, cu(np.arange(len(ref.scale[0]))), *(cu(c, torch.int8) for c in ref.codes),
                   *(cu(s, torch.float32) for s in ref.scale))
        _, out = run_attention(cache, ref, table, [50], [4], "f32", 2, rng)
        assert not bool(out[:4].any())


def test_nan_stays_where_it_is_seen():
    """A page of NaN scale spoils the rows that see it; pages behind the last
    position, other sequences' and other heads' pages do not matter."""
    rng = np.random.default_rng(15)
    lens = [40, 40]
    cache, ref, table = batch(rng, 2, 64, 16, lens)
    with cache:
        nan = np.float32("nan")
        seen = [int(x) for x in table[0, :3]] + [int(x) for x in table[1, :3]]
        for p in range(len(ref.scale[0])):
            if p not in seen:
                ref.scale[0][p] = ref.scale[1][p] = nan  # nobody's pages
        ref.scale[1][table[0, 2], 1] = nan  # sequence 0, head 1, positions 32..
        cache.load(0, cu(np.arange(len(ref.scale[0]))), *(cu(c, torch.int8) for c in ref.codes),
                   *(cu(s, torch.float32) for s in ref.scale))
        q = torch.tensor(rng.standard_normal((24, 2, 64)), device="cuda", dtype=torch.float32)
        out = cache.attention(0, q, cu([0, 20, 24]), cu(lens), cu(table))
        nans = torch.isnan(out).any(-1).cpu().numpy()
        want = np.zeros((24, 2), bool)
        want[12:20, 1] = True  # rows at positions 32..39
        assert np.array_equal(nans, want)
        # a query that is not finite spoils its own row and head
        q[3, 0, 5] = float("inf")
        out = cache.attention(0, q, cu([0, 20, 24]), cu(lens), cu(table))
        want[3, 0] = True
        assert np.array_equal(torch.isnan(out).any(-1).cpu().numpy(), want)


def test_bad_pages_and_lengths_are_skipped_and_reported():
    rng = np.random.default_rng(16)
    lens = [40, 40, 40]
    cache, ref, table = batch(rng, 1, 64, 16, lens)
    with cache:
        q = torch.tensor(rng.standard_normal((3, 2, 64)), device="cuda", dtype=torch.float32)
        good = cache.attention(0, q, cu([0, 1, 2, 3]), cu(lens), cu(table))
        for id_ in (-1, len(ref.scale[0]), 2**31 - 1):
            broken = table.copy()
            broken[1, 1] = id_
            out = cache.attention(0, q, cu([0, 1, 2, 3]), cu(lens), cu(broken))
            assert cache.status() == _lib.TQ_KV_STATUS_PAGE
            assert torch.equal(out[[0, 2]], good[[0, 2]])
        out = torch.full_like(q, 9)
        cache.attention(0, q, cu([0, 1, 2, 3]), cu([40, -1, 40]), cu(table), out=out)
        assert cache.status() == _lib.TQ_KV_STATUS_LENGTH
        assert torch.equal(out[[0, 2]], good[[0, 2]]) and bool((out[1] == 9).all())
        cache.attention(0, q, cu([0, 1, 2, 3]), cu([40, 1000, 40]), cu(table), out=out)
        assert cache.status() == _lib.TQ_KV_STATUS_TABLE and bool((out[1] == 9).all())
        cache.attention(0, q, cu([0, 2, 1, 3]), cu(lens), cu(table), out=out)
        assert cache.status() == _lib.TQ_KV_STATUS_LENGTH
        cache.attention(0, q, cu([0, 1, 2, 99]), cu(lens), cu(table), out=out)
        assert cache.status() == _lib.TQ_KV_STATUS_LENGTH


def test_strided_queries_and_outputs():
    rng = np.random.default_rng(17)
    lens, new = [70, 9], [3, 1]
    cache, ref, table = batch(rng, 2, 64, 32, lens)
    with cache:
        dense = torch.tensor(rng.standard_normal((4, 6, 64)), device="cuda").to(torch.bfloat16)
        starts = cu([0, 3, 4])
        want = cache.attention(0, dense, starts, cu(lens), cu(table))
        for offset, width in ((0, 512), (3, 517)):
            rows = torch.zeros((4, width), device="cuda", dtype=torch.bfloat16)
            rows[:, offset:offset + 384] = dense.view(4, -1)
            res = torch.full((4, width), 7, device="cuda", dtype=torch.bfloat16)
            out = res[:, offset:offset + 384].unflatten(1, (6, 64))
            cache.attention(0, rows[:, offset:offset + 384].unflatten(1, (6, 64)), starts, cu(lens), cu(table), out=out)
            assert torch.equal(out, want) and bool((res[:, offset + 384:] == 7).all())
            assert bool((res[:, :offset] == 7).all())


def prompts(rng, dtype="f32", group=4):
    """Three sequences with rows for the tensor-memory kernel, one without."""
    lens, new = [300, 140, 50, 200], [100, 140, 3, 33]
    cache, ref, table = batch(rng, 2, 64, 16, lens)
    starts = np.concatenate([[0], np.cumsum(new)])
    q = torch.tensor(rng.standard_normal((starts[-1], 2 * group, 64)), device="cuda").to(DT[dtype])
    return cache, ref, widen(table, len(q), 2 * group, 64, 16), lens, starts, q


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_prompts_nan_stays_where_it_is_seen(dtype):
    rng = np.random.default_rng(22)
    cache, ref, table, lens, starts, q = prompts(rng, dtype)
    with cache:
        nan = np.float32("nan")
        good = cache.attention(0, q, cu(starts), cu(lens), cu(table))
        used = set(table[table >= 0].tolist())
        for p in range(len(ref.scale[0])):
            if p not in used:
                ref.scale[0][p] = ref.scale[1][p] = nan  # nobody's pages
        ref.scale[1][table[0, 15], 1] = nan  # sequence 0, head 1, positions 240 to 255: its tokens 40 and later
        ref.scale[0][table[3, 11], 0] = nan  # sequence 3, head 0, positions 176 to 191: its tokens 9 and later
        cache.load(0, cu(np.arange(len(ref.scale[0]))), *(cu(c, torch.int8) for c in ref.codes),
                   *(cu(s, torch.float32) for s in ref.scale))
        want = np.zeros((len(q), 8), bool)
        want[40:100, 4:] = True
        want[starts[3] + 9:, :4] = True
        q[7, 2, 5] = float("inf")  # a query that is not finite spoils its own row
        want[7, 2] = True
        out = cache.attention(0, q, cu(starts), cu(lens), cu(table))
        assert np.array_equal(torch.isnan(out).any(-1).cpu().numpy(), want)
        clean = torch.tensor(~want, device="cuda")
        # the rest is as it was but for p's rounding to float16 (2^-12 of the largest value either way, where a
        # row's largest score is known in another order) and the output's (2^-12 either way)
        assert float((out.float() - good.float())[clean].abs().max()) <= 4 * 2.0**-12 * float(good.float().abs().max())


def test_prompts_bad_pages_and_lengths_are_skipped_and_reported():
    rng = np.random.default_rng(23)
    cache, ref, table, lens, starts, q = prompts(rng)
    with cache:
        good = cache.attention(0, q, cu(starts), cu(lens), cu(table))
        others = torch.ones(len(q), dtype=torch.bool, device="cuda")
        others[100:240] = False
        for id_ in (-1, len(ref.scale[0]), 2**31 - 1):
            broken = table.copy()
            broken[1, 4] = id_
            out = cache.attention(0, q, cu(starts), cu(lens), cu(broken))
            assert cache.status() == _lib.TQ_KV_STATUS_PAGE
            assert torch.equal(out[others], good[others])
            assert torch.equal(out[100:164], good[100:164])  # they do not see it
        # without sequence 1 the work is cut elsewhere: the others' sums are joined in another order
        want, mag, qk, top_v = ref.attention(np_(q), starts, lens, table, 64**-0.5)
        tol = bound(want, mag, qk, top_v, "f32", 64, 4, 300, [], many=True)
        for length, bit in ((-1, _lib.TQ_KV_STATUS_LENGTH), (2**30, _lib.TQ_KV_STATUS_TABLE)):
            out = torch.full_like(q, 9)
            cache.attention(0, q, cu(starts), cu([300, length, 50, 200]), cu(table), out=out)
            assert cache.status() == bit and bool((out[100:240] == 9).all())
            assert np.all((np.abs(np_(out) - want) <= tol)[np_(others)])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_prompts_strided(dtype):
    rng = np.random.default_rng(24)
    cache, ref, table, lens, starts, q = prompts(rng, dtype)
    with cache:
        args = (cu(starts), cu(lens), cu(table))
        want = cache.attention(0, q, *args)
        assert torch.equal(cache.attention(0, q, *args), want)  # the same bits
        for offset, width in ((0, 1024), (3, 517)):
            rows = torch.zeros((len(q), width), device="cuda", dtype=q.dtype)
            rows[:, offset:offset + 512] = q.view(len(q), -1)
            res = torch.full((len(q), width), 7, device="cuda", dtype=q.dtype)
            out = res[:, offset:offset + 512].unflatten(1, (8, 64))
            cache.attention(0, rows[:, offset:offset + 512].unflatten(1, (8, 64)), *args, out=out)
            assert torch.equal(out, want) and bool((res[:, offset + 512:] == 7).all())
            assert bool((res[:, :offset] == 7).all())


def test_prompts_in_graphs_and_streams_side_by_side():
    rng = np.random.default_rng(25)
    cache, ref, table, lens, starts, q = prompts(rng, "bf16")
    with cache:
        args = (cu(starts), cu(lens), cu(table))
        want = cache.attention(0, q, *args)
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = [cache.attention(0, q, *args) for _ in range(2)]
            graphs.append((g, out, torch.cuda.Stream()))
        for _ in range(5):
            for g, _, st in graphs:
                with torch.cuda.stream(st):
                    g.replay()
            eager = cache.attention(0, q, *args)
            torch.cuda.synchronize()
            assert torch.equal(eager, want)
            assert all(torch.equal(x, want) for _, out, _ in graphs for x in out)
            for _, out, _ in graphs:
                for x in out:
                    x.zero_()


@pytest.mark.parametrize("tiny", [1e-44, 1e-38, 2e-30])
def test_prompts_of_tiny_values(tiny):
    """Pages whose value scale is next to nothing beside ordinary ones, and
    nothing else in a whole sequence: no overflow of its inverse."""
    rng = np.random.default_rng(26)
    cache, ref, table, lens, starts, q = prompts(rng)
    with cache:
        for i in table[0, 3:9]:
            ref.scale[1][i] = tiny
        for i in table[1][table[1] >= 0]:
            ref.scale[1][i] = tiny
        cache.load(0, cu(np.arange(len(ref.scale[0]))), *(cu(c, torch.int8) for c in ref.codes),
                   *(cu(s, torch.float32) for s in ref.scale))
        want, mag, qk, top_v = ref.attention(np_(q), starts, lens, table, 64**-0.5)
        tol = bound(want, mag, qk, top_v, "f32", 64, 4, 300, [], many=True)
        for rows in (table, table[:, :30]):  # the tensor-memory kernel, the small one
            out = np_(cache.attention(0, q, cu(starts), cu(lens), cu(rows)))
            # values of scales below 2^-92 may count as 0: 127 * 2^-92 at most
            assert np.all(np.abs(out - want) <= tol + 127 * 2.0**-92)


def test_loaded_scales_are_magnitudes():
    with KVCache(1, 1, 8, 16, 3) as cache:
        codes = torch.ones((3, 16, 1, 8), dtype=torch.int8, device="cuda")
        a, b = cu([[-1.0], [float("inf")], [2.0]], torch.float32), cu([[1.0], [-0.0], [float("-inf")]], torch.float32)
        cache.load(0, cu([0, 1, 2]), codes, codes, a, b)
        _, _, ks, vs = cache.save(0, cu([0, 1, 2]))
        assert torch.isnan(ks[:, 0]).tolist() == [True, True, False] and float(ks[2]) == 2
        assert torch.isnan(vs[:, 0]).tolist() == [False, False, True] and float(vs[0]) == 1 and float(vs[1]) == 0
        cache.check()


def test_offsets_beyond_32_bits():
    rng = np.random.default_rng(18)
    n_pages, n_kv, hd, page = 40000, 8, 128, 128  # 5.2 GB of keys
    with KVCache(1, n_kv, hd, page, n_pages) as cache:
        x = torch.tensor(rng.standard_normal((2, 200, n_kv, hd)), device="cuda").to(torch.bfloat16)
        ids = [n_pages - 1, n_pages - 3]
        slots = [ids[p // page] * page + p % page for p in range(200)]
        cache.store(0, x[0], x[1], i64(slots))
        small = kvref.Ref(n_kv, hd, page, 2)
        small.store(np_(x[0]), np_(x[1]), np.arange(200))
        k, v, ks, vs = cache.save(0, cu(ids))
        assert np.array_equal(k.cpu().numpy(), small.codes[0]) and np.array_equal(v.cpu().numpy(), small.codes[1])
        q = torch.tensor(rng.standard_normal((2, n_kv, hd)), device="cuda", dtype=torch.float32)
        out = cache.attention(0, q, cu([0, 2]), cu([200]), cu([ids]))
        want, mag, qk, top_v = small.attention(np_(q), [0, 2], [200], np.array([[0, 1]]), hd**-0.5)
        assert np.all(np.abs(np_(out) - want) <= bound(want, mag, qk, top_v, "f32", hd, 1, 200, [2]))
        cache.check()


# ---- together ---------------------------------------------------------------------------

def test_a_serving_run():
    """Requests join, decode and leave; plan, store and attention of every step
    against the restatement."""
    rng = np.random.default_rng(19)
    n, page, n_pages, n_kv, hd, n_q = 5, 16, 60, 2, 64, 6
    with KVCache(1, n_kv, hd, page, n_pages) as cache:
        ref = kvref.Ref(n_kv, hd, page, n_pages)
        random_pages(cache, ref, rng)
        lens, table = cu(np.zeros(n)), cu(np.full((n, 12), -1))
        free, count, starts = cu(rng.permutation(n_pages)), cu([n_pages]), cu(np.zeros(n + 1))
        slots = i64(np.full(200, -1))
        for step in range(12):
            held = np_(lens)
            added = np.where(held == 0, rng.integers(0, 40, n), 1)
            T = int(added.sum())
            w_starts, w_lens, w_slots, w_table, _ = kvref.plan(held, added, np_(table), np_(free)[:int(count)], page)
            cache.plan(lens, cu(added), table, free, count, starts, lens, slots)
            assert np.array_equal(np_(slots)[:T], w_slots) and np.array_equal(np_(table), w_table)
            q, k, v = (torch.tensor(rng.standard_normal((200, h, hd)), device="cuda", dtype=torch.float32)
                       for h in (n_q, n_kv, n_kv))
            slots[T:] = -1
            cache.store(0, k, v, slots)
            ref.store(np_(k)[:T], np_(v)[:T], w_slots)
            out = cache.attention(0, q, starts, lens, table)
            want, mag, qk, top_v = ref.attention(np_(q)[:T], w_starts, w_lens, w_table, hd**-0.5)
            assert np.all(np.abs(np_(out)[:T] - want) <= bound(want, mag, qk, top_v, "f32", hd, 3, 60, list(added)))
            if step % 4 == 3:
                cache.release(cu((rng.random(n) < 0.5).astype(int)), lens, table, free, count)
        cache.check()
        codes_equal(cache, ref, np.arange(n_pages))


def graph_step(cache, state, n_q, dtype):
    """One decode step of every request on static buffers."""
    cache.plan(state["lens"], state["one"], state["table"], state["free"], state["count"], state["starts"],
               state["lens"], state["slots"])
    cache.store(0, state["k"], state["v"], state["slots"])
    return cache.attention(0, state["q"], state["starts"], state["lens"], state["table"])


def step_state(rng, n, page, n_pages, n_kv, n_q, hd, first):
    f = lambda h: torch.tensor(rng.standard_normal((n, h, hd)), device="cuda", dtype=torch.float32)  # noqa: E731
    width = n_pages // n
    table = np.arange(n * width).reshape(n, width)
    s = dict(lens=cu(first), one=cu([1] * n), table=cu(table), starts=cu(np.zeros(n + 1)), slots=i64(np.zeros(n)),
             free=cu([0] * 4), count=cu([0]), q=f(n_q), k=f(n_kv), v=f(n_kv))
    # the free list hands out each request's own next page: rows are laid out beforehand
    need = [kvref.pages(v, page) for v in first]
    order = []
    lens = list(first)
    for _ in range(80):
        for i in range(n):
            if lens[i] % page == 0 and need[i] < width:
                order.append(table[i, need[i]])
                need[i] += 1
            lens[i] += 1
    s["free"], s["count"] = cu(order[::-1]), cu([len(order)])
    return s


def test_captured_steps_replay_like_eager_ones():
    """The whole step in one graph: lengths, tables and the free count move on
    the device; two graphs of two caches replay at once on two streams."""
    rng = np.random.default_rng(20)
    n, page, n_kv, n_q, hd, steps = 4, 16, 2, 8, 64, 30
    first = [0, 15, 16, 100]
    made = []
    for _ in range(2):
        seed = int(rng.integers(1 << 30))
        eager, graphed = (KVCache(1, n_kv, hd, page, 64) for _ in range(2))
        es, gs = (step_state(np.random.default_rng(seed), n, page, 64, n_kv, n_q, hd, first) for _ in range(2))
        made.append((eager, graphed, es, gs))
    side = [torch.cuda.Stream() for _ in made]
    graphs, outs = [], []
    for (eager, graphed, es, gs), st in zip(made, side):
        st.wait_stream(torch.cuda.current_stream())
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(graph_step(graphed, gs, n_q, torch.float32))
        graphs.append(g)
    for step in range(steps):
        for g, st in zip(graphs, side):
            with torch.cuda.stream(st):
                g.replay()
        for st in side:
            st.synchronize()
        for (eager, graphed, es, gs), out in zip(made, outs):
            want = graph_step(eager, es, n_q, torch.float32)
            assert torch.equal(out, want), step
            assert all(torch.equal(es[k], gs[k]) for k in ("lens", "table", "count", "starts", "slots"))
    for eager, graphed, _, _ in made:
        eager.check()
        graphed.check()
        eager.free()
        graphed.free()


def test_streams_run_side_by_side():
    rng = np.random.default_rng(21)
    lens = [5000, 77]
    cache, ref, table = batch(rng, 2, 64, 64, lens)
    with cache:
        qs = [torch.tensor(rng.standard_normal((2, 8, 64)), device="cuda", dtype=torch.float32) for _ in range(2)]
        args = (cu([0, 1, 2]), cu(lens), cu(table))
        want = [cache.attention(0, q, *args) for q in qs]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in qs]
        got = [[], []]
        for _ in range(20):
            for i, st in enumerate(streams):
                if len(got[i]) % 2:
                    got[i].append(cache.attention(0, qs[i], *args, stream=st))
                else:
                    with torch.cuda.stream(st):
                        got[i].append(cache.attention(0, qs[i], *args))
        torch.cuda.synchronize()
        assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


# ---- refusals ---------------------------------------------------------------------------

def test_wrong_tensors_are_refused():
    with KVCache(1, 2, 64, 16, 4) as cache:
        x = torch.zeros((3, 2, 64), device="cuda")
        slots, starts, lens, table = i64([0, 1, 2]), cu([0, 3]), cu([3]), cu([[0]])
        for bad in (x.cpu(), x.double(), x[:, :1], x[..., :32], x.transpose(1, 2), x[0], x[..., ::2]):
            with pytest.raises(ValueError, match="tensai: k"):
                cache.store(0, bad, x, slots)
        with pytest.raises(ValueError, match="same tokens"):
            cache.store(0, x, x[:2], slots)
        with pytest.raises(ValueError, match="slots"):
            cache.store(0, x, x, slots[:2])
        with pytest.raises(ValueError, match="slots"):
            cache.store(0, x, x, slots.int())
        with pytest.raises(ValueError, match="starts"):
            cache.attention(0, x, starts[:1], lens, table)
        with pytest.raises(ValueError, match="table"):
            cache.attention(0, x, starts, lens, table.long())
        with pytest.raises(ValueError, match="table"):
            cache.attention(0, x, starts, lens, cu([[0], [1]]))
        with pytest.raises(ValueError, match="out"):
            cache.attention(0, x, starts, lens, table, out=torch.zeros_like(x).half())
        with pytest.raises(TensaiError, match="overlaps"):
            cache.attention(0, x, starts, lens, table, out=x)
        with pytest.raises(TensaiError, match="do not share"):
            cache.attention(0, torch.zeros((3, 3, 64), device="cuda"), starts, lens, table)
        with pytest.raises(TensaiError, match="layer 1"):
            cache.store(1, x, x, slots)
        with pytest.raises(TensaiError, match="scale"):
            cache.attention(0, x, starts, lens, table, scale=float("nan"))
        with pytest.raises(TensaiError, match="workspace"):
            cache.attention(0, x, starts, lens, table, workspace=torch.zeros(4096, dtype=torch.uint8, device="cuda"))
        space = cache.workspace()
        with pytest.raises(TensaiError, match="workspace overlaps"):
            cache.attention(0, x, starts, lens, table, workspace=space, out=space[4096:4096 + 1536].view(torch.float32).view_as(x))
        for name, args in (("store", (0, x.data_ptr(), x.data_ptr(), 0, 128, 128, slots.data_ptr() + 4, 3)),
                           ("store", (0, x.data_ptr() + 2, x.data_ptr(), 0, 128, 128, slots.data_ptr(), 2)),
                           ("save", (0, lens.data_ptr() + 1, 1, x.data_ptr(), x.data_ptr(), x.data_ptr(), x.data_ptr()))):
            with pytest.raises(TensaiError, match="not aligned"):
                _lib.check(getattr(cache._L, f"tq_kv_{name}_dev")(cache._h, *args, 0))
        c, f, k = cu([0]), cu([1, 2]), cu([2])
        with pytest.raises(TensaiError, match="overlap"):
            cache.plan(c, cu([1]), table, f, k, cu([0, 0]), k, slots)
        with pytest.raises(TensaiError, match="overlap"):
            cache.release(c, c, table, f, k)
        with pytest.raises(ValueError, match="pages"):
            cache.read(0, i64([0]))
        cache.check()
        empty = cache.attention(0, x[:0], starts * 0, lens, table)
        assert empty.shape == (0, 2, 64)
    with pytest.raises(TensaiError, match="freed cache"):
        cache.store(0, x, x, slots)
    cache.free()  # again: nothing


def test_a_failed_allocation_is_an_error():
    L = _lib.load()
    for n in (1, 2, 4):
        _lib.check(L.tq_debug_fail_allocs(n))
        with pytest.raises(TensaiError) as e:
            KVCache(2, 1, 64, 16, 4)
        assert e.value.code == _lib.TQ_ERR_NOMEM
        _lib.check(L.tq_debug_fail_allocs(0))
