"""The paged 8-bit key/value cache: its bookkeeping, its store and the attention that reads it.

Three operators of one serving step, each as a user's program calls it:

  plan       from the cached and the added length of each request: the pages that the step needs, taken
             from the free list into the block tables, and the slot of each new token;
  store      new keys and values into their slots, as int8 codes with one float32 scale for each page and
             head (codes that a page holds already are rounded again when its scale grows);
  attention  of each request's new tokens over its cached ones, causal, grouped heads, float32, float16 or
             bfloat16 queries, from one token a request to whole prompts.

`own` false: the plain form, elementary torch operations. `own` true: tensai_b200.KVCache.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"


# ---- cases ---------------------------------------------------------------------------------------------

def listed():
    return [
        # a small server's step: eight requests, one token each
        dict(name="plan-8", op="plan", n=8, page=64, max_cached=2048, long_share=0.0, max_added=1, spread=1),
        # a loaded server's step: most requests decode, a twentieth bring a prompt or a piece of one
        dict(name="plan-1024", op="plan", n=1024, page=16, max_cached=4096, long_share=0.05, max_added=2048, spread=2),
        # a decode step's keys and values of one layer (the 7B decoder's heads)
        dict(name="store-decode-32", op="store", n=32, n_kv=4, hd=128, page=64, dtype="bf16", max_cached=2048,
             max_added=1, spread=3),
        # prompts of one layer, some of them continuing a page
        dict(name="store-prompt-bf16", op="store", n=6, n_kv=4, hd=128, page=64, dtype="bf16", max_cached=512,
             max_added=4096, spread=4),
        # the small decoder's heads in float32, short prompts, small pages
        dict(name="store-prompt-f32", op="store", n=9, n_kv=12, hd=64, page=16, dtype="f32", max_cached=100,
             max_added=400, spread=5),
        # the decode step of one request at the end of its context: latency
        dict(name="decode-1-f32", op="attention", n=1, n_q=28, n_kv=4, hd=128, page=64, dtype="f32", max_len=2559,
             mode="decode", queries=1, spread=6),
        # a batch of small-decoder requests (one query head for each KV head)
        dict(name="decode-48-f16", op="attention", n=48, n_q=12, n_kv=12, hd=64, page=16, dtype="f16", max_len=1024,
             mode="decode", queries=1, spread=7),
        # a server's batch of very different lengths, empty rows among them
        dict(name="decode-64-bf16", op="attention", n=64, n_q=28, n_kv=4, hd=128, page=64, dtype="bf16",
             max_len=16384, mode="decode", queries=1, spread=8),
        # two long documents
        dict(name="decode-long-bf16", op="attention", n=2, n_q=28, n_kv=4, hd=128, page=128, dtype="bf16",
             max_len=262144, mode="decode", queries=1, spread=9),
        # a 64-row prompt chunk of the float32 engine
        dict(name="chunk-64-f32", op="attention", n=1, n_q=28, n_kv=4, hd=128, page=64, dtype="f32", max_len=2048,
             mode="prompt", queries=64, spread=10),
        # whole prompts
        dict(name="prompt-bf16", op="attention", n=4, n_q=28, n_kv=4, hd=128, page=64, dtype="bf16", max_len=4096,
             mode="prompt", queries=4096, spread=11),
        # prompt pieces and decoding requests in one call
        dict(name="mixed-f16", op="attention", n=24, n_q=32, n_kv=8, hd=128, page=32, dtype="f16", max_len=6000,
             mode="mixed", queries=700, spread=21),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["plan", "store", "attention", "attention"])
    c = dict(op=op, page=rng.choice([16, 32, 64, 128]), spread=rng.randrange(1 << 30))
    if op == "plan":
        c |= dict(n=_log(rng, 1, 1024), max_cached=_log(rng, 1, 4096), long_share=rng.choice([0.0, 0.02, 0.05]),
                  max_added=_log(rng, 1, 2048))
        return c
    c |= dict(n_kv=rng.choice([1, 2, 4, 5, 8, 12]), hd=rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 256]),
              dtype=rng.choice(["f32", "f16", "bf16", "bf16"]))
    if op == "store":
        if rng.random() < 0.5:
            c |= dict(n=_log(rng, 1, 256), max_cached=_log(rng, 1, 2048), max_added=1)
        else:
            c |= dict(n=_log(rng, 1, 8), max_cached=_log(rng, 1, 512), max_added=_log(rng, 2, 2048))
        return c
    group = rng.choice([1, 1, 2, 3, 4, 6, 7, 8, 16])
    c["n_q"] = c["n_kv"] * group
    c["mode"] = rng.choice(["decode", "decode", "prompt", "mixed"])
    width = c["n_kv"] * c["hd"]  # the cost is kept under the largest listed cases'
    if c["mode"] == "decode":
        c["n"] = _log(rng, 1, 128)
        c["max_len"] = _log(rng, 1, max(64, min(100000, 24_000_000 // (c["n"] * max(width, 512) // 16))))
        c["queries"] = rng.choice([1, 1, 1, 2, 5])
    else:
        c["n"] = _log(rng, 1, 8)
        c["max_len"] = _log(rng, 2, min(12000, int(math.sqrt(5e10 / (2 * c["n"] * c["n_q"] * c["hd"])))))
        c["queries"] = _log(rng, 2, c["max_len"] + 1)
    return c


# ---- the lengths of a case (of the case alone: values come from the seed) ----------------------------------

def _lengths(c):
    """(cached, added) of each request."""
    rng = random.Random(c["spread"])
    cached, added = [], []
    if c["op"] in ("plan", "store"):
        for i in range(c["n"]):
            cached.append(0 if rng.random() < 0.1 else _log(rng, 1, c["max_cached"]))
            if c["op"] == "plan":
                a = rng.randint(1, c["max_added"]) if rng.random() < c["long_share"] else int(rng.random() > 0.05)
            else:
                a = _log(rng, max(1, c["max_added"] // 16), c["max_added"])
            added.append(a)
        if sum(added) == 0:
            added[0] = 1
        return cached, added
    for i in range(c["n"]):
        total = c["max_len"] if i == 0 else _log(rng, 1, c["max_len"])
        if c["mode"] == "decode":
            new = rng.randint(1, c["queries"])
            if i >= 4 and rng.random() < 0.05:
                total, new = 0, rng.randint(0, 1)  # a row of the batch that holds no request
        elif c["mode"] == "prompt" or rng.random() < 0.25:
            new = min(total, c["queries"] if i == 0 else _log(rng, 1, c["queries"]))
        else:
            new = 1
        cached.append(max(0, total - new))
        added.append(new)
    return cached, added


def _pages(length, page):
    return -(-length // page)


def _prefix(counts):
    out = [0]
    for v in counts:
        out.append(out[-1] + v)
    return out


# ---- inputs ------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 7919 + 17)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _tables(lengths, page, width, g, spare=0):
    """Random pages of one pool for every request: (table with -1 behind each row's end, pages of the pool, the
    pool's other pages)."""
    need = [_pages(v, page) for v in lengths]
    n_pages = sum(need) + spare
    order = torch.randperm(n_pages, device=DEV, generator=g).to(torch.int32)
    col = torch.arange(width, device=DEV)[None, :]
    start = torch.tensor(_prefix(need)[:-1], device=DEV)[:, None]
    used = col < torch.tensor(need, device=DEV)[:, None]
    table = torch.where(used, order[(start + col).clamp(max=n_pages - 1)], torch.full_like(order[:1], -1))
    return table.contiguous(), n_pages, order[sum(need):].contiguous()


def _codes(shape, g):
    """int8 codes as quantized activations have them: bell-shaped, the largest of a page near 127."""
    out = torch.empty(shape, dtype=torch.int8, device=DEV)
    flat = out.view(-1)
    step = 1 << 27
    for at in range(0, flat.numel(), step):
        part = flat[at:at + step]
        part.copy_((torch.randn(part.shape, device=DEV, generator=g) * 34).round().clamp(-127, 127))
    return out


def prepare(case, seed):
    c, g = case, _gen(seed)
    cached, added = _lengths(c)
    page, s = c["page"], dict(case=c, page=c["page"])
    if c["op"] == "plan":
        width = max(_pages(a + b, page) for a, b in zip(cached, added)) + 1
        grown = sum(_pages(a + b, page) - _pages(a, page) for a, b in zip(cached, added))
        table, n_pages, free = _tables(cached, page, width, g, spare=grown + 37)
        s |= dict(cached=_i32(cached), added=_i32(added), table=table, free_pages=free, free_count=_i32([len(free)]),
                  starts=torch.zeros(c["n"] + 1, dtype=torch.int32, device=DEV),
                  lens=torch.zeros(c["n"], dtype=torch.int32, device=DEV),
                  slots=torch.zeros(sum(added), dtype=torch.int64, device=DEV),
                  free_left=torch.zeros(1, dtype=torch.int32, device=DEV))
        if own:
            from tensai_b200 import KVCache
            s["cache"] = KVCache(n_layer=1, n_kv=1, hd=64, page=page, n_pages=n_pages)
        return s
    lens = [a + b for a, b in zip(cached, added)]
    n_kv, hd, dt = c["n_kv"], c["hd"], DTYPES[c["dtype"]]
    width = max(1, max(_pages(v, page) for v in lens))
    table, n_pages, _ = _tables(lens, page, width, g, spare=1)
    kcodes, vcodes = _codes((n_pages, page, n_kv, hd), g), _codes((n_pages, page, n_kv, hd), g)
    # largest values between about 1 and 8 for keys, 0.25 and 2 for values
    kscale = torch.exp2(torch.rand((n_pages, n_kv), device=DEV, generator=g) * 3) / 127
    vscale = torch.exp2(torch.rand((n_pages, n_kv), device=DEV, generator=g) * 3 - 2) / 127
    T = sum(added)
    starts = _prefix(added)
    if c["op"] == "store":
        at = torch.arange(T, device=DEV)
        start = torch.tensor(starts, device=DEV)
        row = torch.searchsorted(start, at, right=True) - 1
        pos = torch.tensor(cached, device=DEV)[row] + at - start[row]
        ids = table[row, pos // page].long()
        amp = torch.exp2(torch.rand((1, n_kv, hd), device=DEV, generator=g) * 3 - 1)
        s |= dict(slots=ids * page + pos % page, touched=torch.unique(ids).to(torch.int32),
                  k=(torch.randn((T, n_kv, hd), device=DEV, generator=g) * amp).to(dt),
                  v=torch.randn((T, n_kv, hd), device=DEV, generator=g).to(dt))
    else:
        s |= dict(q=(torch.randn((T, c["n_q"], hd), device=DEV, generator=g) * 1.5).to(dt), table=table,
                  starts=_i32(starts), lens=_i32(lens), max_new=max(added), max_len=max(lens))
    if own:
        from tensai_b200 import KVCache
        cache = KVCache(n_layer=1, n_kv=n_kv, hd=hd, page=page, n_pages=n_pages)
        cache.load(0, torch.arange(n_pages, dtype=torch.int32, device=DEV), kcodes, vcodes, kscale, vscale)
        s["cache"] = cache
    else:
        s |= dict(kcodes=kcodes, vcodes=vcodes, kscale=kscale, vscale=vscale)
    return s


# ---- one pass ----------------------------------------------------------------------------------------------

def run(state):
    s, op = state, state["case"]["op"]
    if own:
        cache = s["cache"]
        if op == "plan":
            cache.plan(s["cached"], s["added"], s["table"], s["free_pages"], s["free_count"], s["starts"], s["lens"],
                       s["slots"], free_left=s["free_left"])
            return {k: s[k] for k in ("starts", "lens", "slots", "table", "free_left")}
        if op == "store":
            cache.store(0, s["k"], s["v"], s["slots"])
            k, v = cache.read(0, s["touched"])
            return {"k": k, "v": v}
        return cache.attention(0, s["q"], s["starts"], s["lens"], s["table"])
    if op == "plan":
        return _plan(s)
    if op == "store":
        k, s["kcodes"], s["kscale"] = _store(s, s["k"], s["kcodes"], s["kscale"])
        v, s["vcodes"], s["vscale"] = _store(s, s["v"], s["vcodes"], s["vscale"])
        return {"k": k, "v": v}
    return _attention(s)


def _plan(s):
    page = s["page"]
    cached, added, table = s["cached"].long(), s["added"].long(), s["table"]
    lens = cached + added
    have, want = (cached + page - 1) // page, (lens + page - 1) // page
    first = torch.cumsum(want - have, 0) - (want - have)
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    grown = (col >= have[:, None]) & (col < want[:, None])
    take = s["free_count"].long() - 1 - (first[:, None] + col - have[:, None])
    table = torch.where(grown, s["free_pages"][take.clamp(0, s["free_pages"].numel() - 1)], table)
    starts = torch.cat([torch.zeros_like(added[:1]), torch.cumsum(added, 0)])
    at = torch.arange(s["slots"].numel(), device=table.device)
    row = torch.searchsorted(starts, at, right=True) - 1
    pos = cached[row] + at - starts[row]
    slots = table[row, pos // page].long() * page + pos % page
    return {"starts": starts.int(), "lens": lens.int(), "slots": slots, "table": table,
            "free_left": s["free_count"] - (want - have).sum().int()}


def _store(s, x, codes, scale):
    """The touched pages' values after the store, and the cache's codes and scales with them."""
    page, touched = s["page"], s["touched"].long()
    ids, off = s["slots"] // page, s["slots"] % page
    at = torch.searchsorted(touched, ids)
    new = torch.zeros((len(touched), page) + x.shape[1:], dtype=torch.float64, device=x.device)
    new[at, off] = x.double()
    fresh = torch.zeros((len(touched), page), dtype=torch.bool, device=x.device)
    fresh[at, off] = True
    row = torch.arange(page, device=x.device)[None, :]
    first = torch.where(fresh, row, torch.full_like(row, page)).amin(1, keepdim=True)
    old = row < first
    was = torch.where(old[:, :1], scale[touched], torch.zeros_like(scale[:1]))
    now = torch.maximum((new.abs().amax((1, 3)) / 127).float(), was)
    q = codes[touched]
    over = torch.where(now > 0, now, torch.ones_like(now)).double()[:, None, :, None]
    kept = (q.double() * was.double()[:, None, :, None] / over).round()
    coded = (new / over).round().clamp(-127, 127)
    q = torch.where(fresh[..., None, None], coded, torch.where(old[..., None, None], kept, q.double())).to(torch.int8)
    codes[touched] = q
    scale[touched] = now
    return q.float() * now[:, None, :, None], codes, scale


def _attention(s):
    c, page = s["case"], s["page"]
    n, n_kv, hd, group = c["n"], c["n_kv"], c["hd"], c["n_q"] // c["n_kv"]
    starts, lens, dev = s["starts"].long(), s["lens"].long(), s["q"].device
    pos = torch.arange(s["max_len"], device=dev)
    ids = s["table"].long()[:, pos // page].clamp(min=0)                                        # [n][L]
    k = s["kcodes"][ids, pos % page].float() * s["kscale"][ids][..., None]                       # [n][L][n_kv][hd]
    at = torch.arange(s["max_new"], device=dev)
    new = starts[1:] - starts[:-1]
    live = at[None, :] < new[:, None]                                                            # [n][Q]
    where = (starts[:-1, None] + at[None, :]).clamp(max=max(0, s["q"].shape[0] - 1))
    q = s["q"][where].float().view(n, len(at), n_kv, group, hd)
    score = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(n, n_kv, -1, hd), k.permute(0, 2, 3, 1)) * hd ** -0.5
    del k
    last = lens[:, None] - new[:, None] + at[None, :]                                            # a query's position
    seen = (pos[None, None, :] <= last[:, :, None]) & (pos[None, None, :] < lens[:, None, None])
    score = score.view(n, n_kv, group, len(at), -1).masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    score = score.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp_()
    total = score.sum(-1, keepdim=True)
    v = s["vcodes"][ids, pos % page].float() * s["vscale"][ids][..., None]
    out = torch.matmul(score.view(n, n_kv, -1, len(pos)), v.permute(0, 2, 1, 3)).view(n, n_kv, group, len(at), hd)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    out = out.permute(0, 3, 1, 2, 4).reshape(n, len(at), n_kv * group, hd)
    return out[live].to(s["q"].dtype)


# ---- what a pass cannot do without -------------------------------------------------------------------------

def work(case):
    c = case
    cached, added = _lengths(c)
    page, T = c["page"], sum(added)
    lens = [a + b for a, b in zip(cached, added)]
    touched = sum(_pages(b, page) - a // page for a, b in zip(cached, lens) if b > a)
    if c["op"] == "plan":
        grown = sum(_pages(b, page) - _pages(a, page) for a, b in zip(cached, lens))
        table = sum(_pages(b, page) - a // page for a, b in zip(cached, lens))
        return {"bytes": 4 * (4 * c["n"] + 3 + grown + table) + 8 * T, "flops": T}
    size = {"f32": 4, "f16": 2, "bf16": 2}[c["dtype"]]
    width = c["n_kv"] * c["hd"]
    if c["op"] == "store":
        # keys and values in, the codes of the tokens out, and the touched pages' values read back
        return {"bytes": 2 * T * width * (size + 1) + 8 * T + 2 * touched * (page * width * 5 + 8 * c["n_kv"]),
                "flops": 4 * T * width}
    rows = [(a, b) for a, b in zip(added, lens) if a and b]
    pairs = sum(sum(max(0, b - i) for i in range(a)) for a, b in rows)
    held = sum(b for _, b in rows)
    tabled = sum(_pages(b, page) for _, b in rows)
    return {"bytes": 2 * held * width + tabled * (8 * c["n_kv"] + 4) + 2 * T * c["n_q"] * c["hd"] * size + 8 * c["n"],
            "flops": 4 * pairs * c["n_q"] * c["hd"]}


# ---- the definition in 64 bits -------------------------------------------------------------------------------

def _plain_prepare(case, seed):
    global own
    kept, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = kept


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = _plain_prepare(case, seed)
    return _exact_store(s) if case["op"] == "store" else _exact_attention(s)


def _exact_store(s):
    page, slots = s["page"], s["slots"].tolist()
    touched = s["touched"].tolist()
    place = {p: i for i, p in enumerate(touched)}
    offsets = [[] for _ in touched]
    tokens = [[] for _ in touched]
    for t, slot in enumerate(slots):
        offsets[place[slot // page]].append(slot % page)
        tokens[place[slot // page]].append(t)
    out = {}
    for name in ("k", "v"):
        pages = []
        for i, p in enumerate(touched):
            x = s[name][tokens[i]].double()
            codes = s[name + "codes"][p].double()
            least = x.abs().amax((0, 2)) / 127.0
            if min(offsets[i]) > 0:
                least = torch.maximum(least, s[name + "scale"][p].double())
            scale = least.float().double()[None, :, None]  # the scale is held in 32 bits
            safe = torch.where(scale == 0, torch.ones_like(scale), scale)
            head = min(offsets[i])
            codes[:head] = torch.round(codes[:head] * s[name + "scale"][p].double()[None, :, None] / safe)
            codes[offsets[i]] = torch.clamp(torch.round(x / safe), -127, 127)
            pages.append(codes * scale)
        out[name] = torch.stack(pages)
    return out


def _exact_attention(s):
    c, page = s["case"], s["page"]
    n_kv, hd, group = c["n_kv"], c["hd"], c["n_q"] // c["n_kv"]
    starts, lens, table = s["starts"].tolist(), s["lens"].tolist(), s["table"].long()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for i, length in enumerate(lens):
        new = starts[i + 1] - starts[i]
        if not new or not length:
            continue
        ids = table[i, :_pages(length, page)]
        for h in range(n_kv):
            k = (s["kcodes"][ids, :, h].double() * s["kscale"][ids, h].double()[:, None, None]).reshape(-1, hd)[:length]
            v = (s["vcodes"][ids, :, h].double() * s["vscale"][ids, h].double()[:, None, None]).reshape(-1, hd)[:length]
            x = s["q"][starts[i]:starts[i + 1], h * group:(h + 1) * group].double()
            for a in range(0, new, 512):
                y = x[a:a + 512]
                z = torch.einsum("qgd,td->qgt", y, k) / math.sqrt(hd)
                row = length - new + a + torch.arange(len(y), device=z.device)
                hidden = torch.arange(length, device=z.device)[None, :] > row[:, None]
                z.masked_fill_(hidden[:, None, :], -math.inf)
                w = torch.nan_to_num(torch.softmax(z, -1), nan=0.0)
                out[starts[i] + a:starts[i] + a + len(y), h * group:(h + 1) * group] = torch.einsum("qgt,td->qgd", w, v)
    return out
