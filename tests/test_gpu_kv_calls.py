"""GPU tests of attention calls over the paged 8-bit cache that are made at once
or on a stream that is not the current one."""
import threading

import numpy as np
import pytest

from tensai_b200 import _lib
from test_gpu_kv import batch, cu, prompts

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def device():
    torch.cuda.init()
    _lib.check(_lib.load().tq_set_device(0))


def test_threads_on_one_stream():
    """Calls of several launches from threads that share a stream, and with it
    the default workspace."""
    rng = np.random.default_rng(51)
    cache, ref, table, lens, starts, q0 = prompts(rng, "bf16")
    with cache:
        args = (cu(starts), cu(lens), cu(table))
        qs = [q0 * (1 + i) for i in range(4)]
        want = [cache.attention(0, q, *args) for q in qs]
        torch.cuda.synchronize()
        start, wrong = threading.Barrier(len(qs)), [0] * len(qs)

        def work(i):
            start.wait()
            got = [cache.attention(0, qs[i], *args) for _ in range(300)]
            torch.cuda.synchronize()
            wrong[i] = sum(not torch.equal(x, want[i]) for x in got)

        threads = [threading.Thread(target=work, args=(i,)) for i in range(len(qs))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert wrong == [0] * len(qs)
        cache.check()
