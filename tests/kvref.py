"""Plain 64-bit restatement of the paged 8-bit cache (numpy): plan, store and
attention, written from their definitions in include/tensai_cuda.h."""
import numpy as np


def pages(length, page):
    return -(-int(length) // page)


def plan(cached, added, table, free, page):
    """(starts, lens, slots, table, free left) of one plan."""
    table, free = table.copy(), list(free)
    starts, lens, slots = [0], [], []
    for i, (c, a) in enumerate(zip(cached, added)):
        for b in range(pages(c, page), pages(c + a, page)):
            table[i, b] = free.pop()
        slots += [int(table[i, p // page]) * page + p % page for p in range(c, c + a)]
        starts.append(starts[-1] + int(a))
        lens.append(int(c + a))
    return np.array(starts), np.array(lens), np.array(slots, np.int64), table, free


class Ref:
    """Codes [n_pages][page][n_kv][hd] and scales [n_pages][n_kv] of keys (0) and values (1)."""

    def __init__(self, n_kv, hd, page, n_pages):
        self.page, self.n_kv, self.hd = page, n_kv, hd
        self.codes = [np.zeros((n_pages, page, n_kv, hd), np.int8) for _ in range(2)]
        self.scale = [np.zeros((n_pages, n_kv), np.float32) for _ in range(2)]

    def store(self, k, v, slots):
        """k, v: float64 arrays [tokens][n_kv][hd] holding the stored type's values."""
        for side, x in enumerate((k, v)):
            t = 0
            while t < len(slots):
                if slots[t] < 0:
                    t += 1
                    continue
                id_, off = divmod(int(slots[t]), self.page)
                run = 1
                while t + run < len(slots) and off + run < self.page and slots[t + run] == slots[t] + run:
                    run += 1
                for h in range(self.n_kv):
                    self._store(side, id_, off, h, x[t:t + run, h])
                t += run

    def _store(self, side, id_, off, h, x):
        codes, was = self.codes[side][id_, :, h], self.scale[side][id_, h]
        most = np.abs(x).max()  # NaN if any is
        now = np.float32(most / 127.0) if np.isfinite(most) else np.float32("nan")
        if off:
            now = now if np.isnan(now) else was if np.isnan(was) else max(now, was)
        if off and not np.isnan(now) and now != was:
            codes[:off] = np.rint(codes[:off].astype(np.float64) * float(was) / float(now))
        new = np.zeros(x.shape) if not now > 0 else np.clip(np.rint(x / float(now)), -127, 127)
        codes[off:off + len(x)] = new
        self.scale[side][id_, h] = now

    def values(self, side, ids):
        return self.codes[side][ids].astype(np.float64) * self.scale[side][ids].astype(np.float64)[:, None, :, None]

    def attention(self, q, starts, lens, table, scale):
        """(out, sum p|v|, largest sum |q k| scale, 127 times the largest value
        scale of the sequence's pages) per row and head, float64."""
        tokens, n_q, hd = q.shape
        group = n_q // self.n_kv
        out, mag = np.zeros(q.shape), np.zeros(q.shape)
        qk, top_v = np.zeros((tokens, n_q)), np.zeros((tokens, n_q))
        for i, length in enumerate(lens):
            new = starts[i + 1] - starts[i]
            if new == 0 or length == 0:
                continue
            ids = table[i, :pages(length, self.page)]
            k = self.values(0, ids).reshape(-1, self.n_kv, hd)[:length]
            v = self.values(1, ids).reshape(-1, self.n_kv, hd)[:length]
            for h in range(n_q):
                kh, vh = k[:, h // group], v[:, h // group]
                x = q[starts[i]:starts[i + 1], h]
                s = x @ kh.T * scale
                seen = np.arange(length)[None, :] <= (length - new + np.arange(new))[:, None]
                s = np.where(seen, s, -np.inf)
                top = s.max(1, keepdims=True)
                p = np.exp(s - np.where(np.isfinite(top), top, 0))
                total = p.sum(1, keepdims=True)
                p = np.where(total > 0, p / np.where(total > 0, total, 1), 0)
                out[starts[i]:starts[i + 1], h] = p @ vh
                mag[starts[i]:starts[i + 1], h] = p @ np.abs(vh)
                qk[starts[i]:starts[i + 1], h] = (np.abs(x) @ np.abs(kh).T).max() * abs(scale)
                top_v[starts[i]:starts[i + 1], h] = 127 * float(self.scale[1][ids, h // group].max())
        return out, mag, qk, top_v
