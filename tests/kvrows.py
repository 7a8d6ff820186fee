"""Row by row restatement of the attention over the paged 8-bit cache (float64),
with what its arithmetic allows from the positions that a row sees alone."""
import numpy as np

import kvref

ZERO = 2.0**-60  # what a page of zeros counts as where the largest weight is looked for


def attend(ref, q, starts, lens, table, scale, dtype_eps, one_piece=False, many=False):
    """(out, tolerance) [tokens][n_q][hd]; a row that sees a scale that is not a
    number is NaN in both. Only what a row sees enters its figures.

    Per position: the score's hd products (22 bits of q, float32 sums that the
    tensor cores may truncate: 2^-22 each) move its weight by twice their error,
    exp2, its argument's rounding and the pieces of p add 2^-19, 2^-11 where p is
    one float16; every addition 2^-22. Held in float16 with the largest weight
    times value scale at 2^13 or more (many rows: 2^10), a weight is off by at
    most 2^-25: 2^-38 (2^-35) of 127 times that position's value scale. Then the
    output's rounding, and its least step."""
    tokens, n_q, hd = q.shape
    group = n_q // ref.n_kv
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for i, length in enumerate(lens):
        new = int(starts[i + 1] - starts[i])
        ids = table[i, :kvref.pages(length, ref.page)]
        k, v = (ref.values(s, ids).reshape(-1, ref.n_kv, hd) for s in range(2))
        c = np.repeat(ref.scale[1][ids].astype(np.float64), ref.page, 0)
        for j in range(new):
            seen = max(0, length - new + j + 1)
            for h in range(n_q) if seen else ():
                x, g = q[starts[i] + j, h], h // group
                kk, vv, cc = k[:seen, g], v[:seen, g], c[:seen, g]
                s = kk @ x * scale
                p = np.exp(s - s.max())
                o = p @ vv / p.sum()
                mag = p @ np.abs(vv) / p.sum()
                qk = (np.abs(kk) @ np.abs(x)).max() * abs(scale)
                top = cc[np.argmax(p * np.maximum(cc, ZERO))]
                rel = 2 * (hd + 16) * 2.0**-22 * qk + (seen + 64) * 2.0**-22 + 2.0**-19 + (2.0**-11 if one_piece else 0)
                floor = seen * (2.0**-35 if many else 2.0**-38) * 127 * top
                out[starts[i] + j, h] = o
                tol[starts[i] + j, h] = mag * rel + floor + np.abs(o) * dtype_eps / 2 * 1.0001
    return out, tol
