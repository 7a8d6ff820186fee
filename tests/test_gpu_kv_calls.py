"""GPU tests of attention calls over the paged 8-bit cache that are made at once
or on a stream that is not the current one."""
import threading
import time

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


def test_a_captured_call_has_its_own_workspace_whatever_stream_is_current():
    """Captured through stream=, with another stream current."""
    rng = np.random.default_rng(52)
    lens = [5000, 77]
    cache, ref, table = batch(rng, 2, 64, 64, lens)
    with cache:
        qs = [torch.tensor(rng.standard_normal((2, 8, 64)), device="cuda", dtype=torch.float32) for _ in range(2)]
        args = (cu([0, 1, 2]), cu(lens), cu(table))
        want = [cache.attention(0, q, *args) for q in qs]
        made, make = [], cache.workspace

        def workspace(stream=None):
            w = make(stream)
            made.append(w.data_ptr())
            return w

        cache.workspace = workspace
        side, other = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        cache.attention(0, qs[0], *args, stream=side)  # the stream's own workspace
        torch.cuda.synchronize()
        assert len(made) == 1
        graphs, outs = [], [torch.empty_like(q) for q in qs]
        for q, out in zip(qs, outs):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                with torch.cuda.stream(other):
                    cache.attention(0, q, *args, out=out, stream=side)
            graphs.append(g)
        assert len(made) == 3 and len(set(made)) == 3
        streams = [torch.cuda.Stream() for _ in graphs]
        for _ in range(20):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
            eager = cache.attention(0, qs[0], *args, stream=side)
            torch.cuda.synchronize()
            assert torch.equal(eager, want[0]) and all(torch.equal(x, y) for x, y in zip(outs, want))
        assert len(made) == 3
        cache.check()


def test_a_stream_is_first_used_in_a_capture():
    """What the capture made stays the graph's: the stream's eager calls begin
    with a workspace of their own."""
    rng = np.random.default_rng(53)
    lens = [5000, 77]
    cache, ref, table = batch(rng, 2, 64, 64, lens)
    with cache:
        q = torch.tensor(rng.standard_normal((2, 8, 64)), device="cuda", dtype=torch.float32)
        args = (cu([0, 1, 2]), cu(lens), cu(table))
        want = cache.attention(0, q, *args)
        side, other, out = torch.cuda.Stream(), torch.cuda.Stream(), torch.empty_like(q)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            with torch.cuda.stream(other):
                cache.attention(0, q, *args, out=out, stream=side)
        assert side.cuda_stream not in cache._spaces
        eager = cache.attention(0, q, *args, stream=side)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager, want) and torch.equal(out, want)
        cache.check()


def test_no_report_is_lost_between_threads():
    """One thread looks at the status all the time, one makes it report, and what
    this one makes it report is seen by one of the two that look."""
    from tensai_b200 import KVCache
    with KVCache(1, 1, 8, 16, 4) as cache:
        stop, seen = threading.Event(), []

        def look():
            while not stop.is_set():
                seen.append(cache.status())

        def noise():
            c, a, t, f, k = cu([-1]), cu([1]), cu([[0]]), cu([0]), cu([1])
            s, ln, sl = cu([0, 0]), cu([0]), torch.zeros(1, dtype=torch.int64, device="cuda")
            st = torch.cuda.Stream()
            while not stop.is_set():
                cache.plan(c, a, t, f, k, s, ln, sl, stream=st)
                st.synchronize()

        threads = [threading.Thread(target=x) for x in (look, noise)]
        for t in threads:
            t.start()
        lost, bad, mine = 0, cu([9]), torch.cuda.Stream()
        try:
            for _ in range(400):
                at = len(seen)
                cache.read(0, bad, stream=mine)
                mine.synchronize()
                for _ in range(20):
                    if cache.status() & _lib.TQ_KV_STATUS_PAGE:
                        break
                    if any(b & _lib.TQ_KV_STATUS_PAGE for b in seen[at:]):
                        break
                else:
                    time.sleep(0.2)  # what the other thread took it may still have to note
                    lost += not any(b & _lib.TQ_KV_STATUS_PAGE for b in seen[at:])
        finally:
            stop.set()
            for t in threads:
                t.join()
        assert lost == 0


def test_freeing_a_cache_that_other_threads_use():
    """Calls under way have made their launches before the memory goes; those behind
    it are errors."""
    from tensai_b200 import KVCache, TensaiError
    for turn in range(10):
        cache = KVCache(1, 1, 64, 16, 64)
        slots, table = torch.arange(256, device="cuda"), cu(np.arange(64)[None, :])
        starts, lens = cu([0, 256]), cu([256])
        started, refused, threads = threading.Barrier(4), [], []

        def work(call):
            x = torch.randn(256, 1, 64, device="cuda")
            space = cache.workspace()
            torch.cuda.synchronize()
            started.wait()
            try:
                for _ in range(100000):
                    if call == "store":
                        cache.store(0, x, x, slots)
                    elif call == "read":
                        cache.read(0, starts[:1])
                    else:
                        cache.attention(0, x, starts, lens, table, workspace=space)
            except TensaiError as e:
                refused.append((call, e.code))

        for call in ("store", "read", "attention"):
            threads.append(threading.Thread(target=work, args=(call,)))
            threads[-1].start()
        started.wait()
        while turn % 2 and cache.status():
            pass
        cache.free()
        for t in threads:
            t.join()
        assert sorted(refused) == [(c, _lib.TQ_ERR_HANDLE) for c in ("attention", "read", "store")]
        torch.cuda.synchronize()
