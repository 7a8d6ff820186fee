"""The Qwen2 engine with its keys and values in the paged 8-bit cache
(tq_qwen_set_cache) against a float64 restatement of the model whose cache is
the restated one (kvref.py): the generated ids, token by token and in chunks."""
import numpy as np
import pytest

import kvref
from oracle import oracle as O
from tensai_b200 import TensaiError, _lib
from tensai_b200.decode import Qwen, synth_tokens
from test_oracle_decode import _deq4

pytestmark = pytest.mark.gpu

TINY = dict(n_layer=2, n_head=4, n_kv=2, d=256, ffn=512, vocab=1000, ctx=192, eps=1e-6, theta=1e6)
WIDE = dict(n_layer=2, n_head=4, n_kv=1, d=512, ffn=512, vocab=1000, ctx=200, eps=1e-6, theta=1e4)
SIGMA = 0.05  # large enough for the attention to matter to the logits


@pytest.fixture(scope="module", autouse=True)
def device():
    import torch
    torch.cuda.init()
    _lib.check(_lib.load().tq_set_device(0))


def restated_logits(cfg, seed, tokens, n_prompt, rows):
    """Logits after each position from n_prompt - 1 on, float64; the prompt in
    chunks of `rows` positions (stored together), then one position at a time."""
    d, ffn, V, nh, nkv = cfg["d"], cfg["ffn"], cfg["vocab"], cfg["n_head"], cfg["n_kv"]
    hd = d // nh
    emb = O.synth((V, d), seed, 1, SIGMA).astype(np.float64)
    lm = _deq4(O.synth((d, V), seed, 2, SIGMA))
    L = []
    for l in range(cfg["n_layer"]):
        s0 = 32 + 16 * l
        L.append([_deq4(O.synth(sh, seed, s0 + i, SIGMA)) for i, sh in enumerate(
            [(d, d), (d, nkv * hd), (d, nkv * hd), (d, d), (d, ffn), (d, ffn), (ffn, d)])])
    n_pages = -(-cfg["ctx"] // 64)
    caches = [kvref.Ref(nkv, hd, 64, n_pages) for _ in L]
    table = np.arange(n_pages)[None, :]

    def rms(v):
        return v / np.sqrt((v * v).mean(-1, keepdims=True) + cfg["eps"])

    def rope(x, pos):  # [rows][heads][hd]
        half = hd // 2
        f = cfg["theta"] ** (-2.0 * np.arange(half) / hd)
        c, s = np.cos(pos[:, None] * f)[:, None], np.sin(pos[:, None] * f)[:, None]
        a, b = x[..., :half], x[..., half:]
        return np.concatenate([a * c - b * s, b * c + a * s], -1)

    out = []
    at = 0
    while at < len(tokens):
        n = min(rows, n_prompt - at) if at < n_prompt else 1
        pos = np.arange(at, at + n)
        x = emb[tokens[at:at + n]]
        for cache, (wq, wk, wv, wo, wg, wu, wd) in zip(caches, L):
            a = rms(x)
            q, k, v = ((a @ w).reshape(n, -1, hd) for w in (wq, wk, wv))
            cache.store(rope(k, pos), v, pos)
            att = cache.attention(rope(q, pos), [0, n], [at + n], table, hd**-0.5)[0]
            x = x + att.reshape(n, d) @ wo
            a = rms(x)
            g = a @ wg
            x = x + (g / (1 + np.exp(-g)) * (a @ wu)) @ wd
        at += n
        if at >= n_prompt:
            out.append(rms(x[-1]) @ lm)
    return out


def check_ids(cfg, seed, prompt, got, rows, slack):
    """Each id is the restated logits' largest, or within slack of it, in units
    of the logits' spread: float32 products (and a key or value that lies next
    to a half step and goes the other way) decide between nearer ones."""
    logits = restated_logits(cfg, seed, np.concatenate([prompt, got[:-1]]).astype(int), len(prompt), rows)
    assert len(logits) == len(got)
    for i, (z, t) in enumerate(zip(logits, got)):
        assert z.max() - z[t] <= slack * z.std(), (i, int(t), int(z.argmax()), float(z.max() - z[t]), float(z.std()))
    return np.mean([int(z.argmax()) == t for z, t in zip(logits, got)])


@pytest.mark.parametrize("cfg,n_prompt,n_gen", [(TINY, 20, 40), (TINY, 1, 70), (WIDE, 63, 30)])
def test_generate_with_the_8_bit_cache(cfg, n_prompt, n_gen):
    prompt = synth_tokens(n_prompt, cfg["vocab"], 3)
    with Qwen(cfg, 3, SIGMA) as m:
        plain = m.generate(prompt, n_gen)
        m.set_cache("int8")
        got = m.generate(prompt, n_gen)
        again = m.generate(prompt, n_gen)
        m.set_cache("float32")
        back = m.generate(prompt, n_gen)
    assert np.array_equal(got, again) and np.array_equal(plain, back)
    # one step of one code of 127 in a key or value moves a logit by far less than this
    assert check_ids(cfg, 3, prompt, got, 1, 0.01) >= 0.9


@pytest.mark.parametrize("rows", [16, 64])
def test_chunked_prompt_with_the_8_bit_cache(rows):
    """Chunks of rows on the tf32 matmul (2e-3 relative per product), stored and
    attended together."""
    prompt = synth_tokens(150, TINY["vocab"], 5)
    with Qwen(TINY, 5, SIGMA) as m:
        m.set_cache("int8")
        m.set_prefill(rows)
        got = m.generate(prompt, 20)
        again = m.generate(prompt, 20)
    assert np.array_equal(got, again)
    check_ids(TINY, 5, prompt, got, rows, 0.1)


def test_the_cache_at_the_end_of_its_context():
    prompt = synth_tokens(100, TINY["vocab"], 7)
    with Qwen(TINY, 7, SIGMA) as m:
        m.set_cache("int8")
        got = m.generate(prompt, TINY["ctx"] - 100 + 1)
        assert len(got) == 93 and m.generate(prompt[:1], 1).shape == (1,)
        with pytest.raises(TensaiError, match="exceed the context"):
            m.generate(prompt, TINY["ctx"] - 100 + 2)
        # sampling keeps working on it
        m.set_sampling(1.0, np.zeros(8))
        assert np.array_equal(m.generate(prompt, 8), got[:8])


def test_set_cache_refuses():
    with Qwen(TINY, 1) as m:
        with pytest.raises(ValueError, match="float32"):
            m.set_cache("int4")
        assert _lib.load().tq_qwen_set_cache(m.handle, 7) == _lib.TQ_ERR_ARG
    assert _lib.load().tq_qwen_set_cache(999, 0) == _lib.TQ_ERR_HANDLE
    with Qwen(TINY, 1) as m:
        want = m.generate([1, 2, 3], 4)
        for n in (1, 3, 7):  # a failed set-up leaves the float32 cache in place
            _lib.check(_lib.load().tq_debug_fail_allocs(n))
            with pytest.raises(TensaiError):
                m.set_cache("int8")
            _lib.check(_lib.load().tq_debug_fail_allocs(0))
            assert np.array_equal(m.generate([1, 2, 3], 4), want)
