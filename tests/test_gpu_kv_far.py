"""GPU tests of the attention over the paged 8-bit cache where scores are so large
that one position takes all the weight."""
import numpy as np
import pytest

import kvref
from tensai_b200 import _lib
from test_gpu_kv import DT, batch, cu, np_, widen

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def device():
    torch.cuda.init()
    _lib.check(_lib.load().tq_set_device(0))


@pytest.mark.parametrize("dtype,group", [("f32", 3), ("bf16", 3), ("f16", 3), ("f16", 12)])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("size", [1e5, 7e5, 1e7, 3e7, 1e9, 1e13, 1e20, 1e30])
def test_large_scores_pick_one_position(dtype, group, many, hd, size):
    """Scores of about `size`: a row whose two largest are more than 2^-9 of the
    largest apart is the value at the larger (both are known to 2^-14, the
    products and sums of 22 bits), within its output's rounding and one part in
    2^18 of weights and sums (one piece: 2^-10)."""
    if many and hd == 256:
        pytest.skip("one kernel")
    rng = np.random.default_rng(61)
    lens, new = [300, 77], ([100, 60] if many else [2, 1])
    cache, ref, table = batch(rng, 2, hd, 16, lens)
    with cache:
        starts = np.concatenate([[0], np.cumsum(new)])
        n_q = 2 * group
        x = rng.standard_normal((starts[-1], n_q, hd))
        q = torch.tensor(x * (1e3 if dtype == "f16" else min(size, 1e20)), device="cuda").to(DT[dtype])
        k = [ref.values(s, np.arange(len(ref.scale[0]))) for s in range(2)]
        unit = np.abs(np.einsum("thd,pd->thp", np_(q)[:4], k[0][:4, 0, 0])).max()
        scale = size / unit
        rows = widen(table, len(q), n_q, hd, 16) if many else table
        out = np_(cache.attention(0, q, cu(starts), cu(lens), cu(rows), scale=scale))
        cache.check()
        assert np.all(np.isfinite(out))
        one = dtype != "f32" and (many or group > 8)
        picked = 0
        for i, length in enumerate(lens):
            ids = table[i, :kvref.pages(length, 16)]
            kk, vv = (k[s][ids].reshape(-1, 2, hd) for s in range(2))
            for j in range(new[i]):
                seen = length - new[i] + j + 1
                for h in range(n_q):
                    t = starts[i] + j
                    s = kk[:seen, h // group] @ np_(q[t, h]) * scale
                    a, b = np.argsort(s)[-2:]
                    if s[b] - s[a] < max(40, 2.0**-9 * abs(s[b])):
                        continue
                    picked += 1
                    want = vv[b, h // group]
                    tol = np.abs(want) * (torch.finfo(DT[dtype]).eps / 2 + 2.0**-18 + (2.0**-10 if one else 0)) + 2.0**-25
                    assert np.all(np.abs(out[t, h] - want) <= tol), (t, h)
        assert picked > 0.5 * len(q) * n_q


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("centre", [2.0**k for k in (18, 20, 21, 22, 23)])
@pytest.mark.parametrize("apart", [1.0, 4.0])
def test_large_scores_that_share_a_row(many, centre, apart):
    """Two positions of different tiles, their scores around `centre` powers of two
    and `apart` apart, so that the second raises the largest. A score's roundings
    (its factor, itself, what is taken off) are at most 2^-22 of it together and
    move a weight by as many powers of two."""
    rng = np.random.default_rng(62)
    new, lens, hd = (60 if many else 1), [300], 64
    cache, ref, table = batch(rng, 1, hd, 16, lens)
    with cache:
        s = np.log(2) * centre + np.array([-apart / 2, apart / 2])
        ref.scale[0][:] = 0
        for at, score in zip((5, 200), s):
            ref.codes[0][table[0, at // 16]] = 0
            ref.codes[0][table[0, at // 16], at % 16] = 127
            ref.scale[0][table[0, at // 16]] = np.float32(score / (64 * 127))
        cache.load(0, cu(np.arange(len(ref.scale[0]))), *(cu(c, torch.int8) for c in ref.codes),
                   *(cu(x, torch.float32) for x in ref.scale))
        q = torch.ones((new, 1, hd), device="cuda")
        rows = widen(table, new, 1, hd, 16) if many else table
        out = np_(cache.attention(0, q, cu([0, new]), cu(lens), cu(rows), scale=1.0))
        cache.check()
        got = [ref.values(0, table[0])[at // 16, at % 16, 0].sum() for at in (5, 200)]
        v = [ref.values(1, table[0])[at // 16, at % 16, 0] for at in (5, 200)]
        share = 1 / (1 + np.exp(got[0] - got[1]))  # of the second
        off = 2 ** min(8.0, 2 * centre * 2.0**-22) - 1
        tol = share * (1 - share) * off * np.abs(v[0] - v[1]) + 2.0**-18 * np.maximum(np.abs(v[0]), np.abs(v[1]))
        assert np.all(np.abs(out - (v[0] + share * (v[1] - v[0]))) <= tol)
