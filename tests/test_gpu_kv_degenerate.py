"""GPU tests of the attention over the paged 8-bit cache: queries, scales and
factors of nothing or next to nothing, on the kernel for many rows as on the
one for few."""
import numpy as np
import pytest

from tensai_b200 import _lib
from test_gpu_kv import DT, batch, cu
from test_gpu_kv_hidden import compare, load

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
LENS = [300, 77, 128]  # position tiles that are full and that are not


@pytest.fixture(scope="module", autouse=True)
def device():
    torch.cuda.init()
    _lib.check(_lib.load().tq_set_device(0))


def case(seed, hd, many):
    rng = np.random.default_rng(seed)
    new = [100, 60, 70] if many else [2, 1, 4]
    cache, ref, table = batch(rng, 2, hd, 16, LENS)
    starts = np.concatenate([[0], np.cumsum(new)])
    return cache, ref, table, starts, rng.standard_normal((starts[-1], 6, hd))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("many", [False, True])
def test_queries_of_nothing_among_others(dtype, hd, many):
    """Whole rows of zeros (a padding token), single heads of zeros, rows of 1e-30."""
    cache, ref, table, starts, x = case(41, hd, many)
    with cache:
        x[starts[0]] = x[starts[1]] = x[-1] = 0
        x[::3, 1] = 0
        x[1::4, 4] *= 1e-30
        q = torch.tensor(x, device="cuda").to(DT[dtype])
        compare(cache, ref, q, starts, LENS, table, dtype, many=many)
        cache.check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("q_scale", [0.0, 1e-30, 1e-4, 30.0])
def test_magnitudes_of_queries(dtype, many, q_scale):
    cache, ref, table, starts, x = case(42, 64, many)
    with cache:
        q = torch.tensor(x * q_scale, device="cuda").to(DT[dtype])
        compare(cache, ref, q, starts, LENS, table, dtype, many=many)
        compare(cache, ref, q, starts, LENS, table, dtype, many=many, scale=0.0)
        cache.check()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("many", [False, True])
def test_keys_of_zeros(dtype, many):
    """Pages of zero key scale, some under the causal mask, with queries of every
    size; then no key at all, and no value."""
    cache, ref, table, starts, x = case(43, 64, many)
    with cache:
        for i in range(3):
            ids = table[i][table[i] >= 0]
            ref.scale[0][ids[::2]] = 0
        load(cache, ref)
        x[::5] = 0
        x[1::5] *= 1e-12
        q = torch.tensor(x, device="cuda").to(DT[dtype])
        compare(cache, ref, q, starts, LENS, table, dtype, many=many)
        ref.scale[0][:] = 0
        load(cache, ref)
        compare(cache, ref, q, starts, LENS, table, dtype, many=many)
        ref.scale[1][:] = 0
        load(cache, ref)
        out = cache.attention(0, q, cu(starts), cu(LENS), cu(table))
        assert not bool(out.any())
        compare(cache, ref, q, starts, LENS, table, dtype, many=many)
        cache.check()
