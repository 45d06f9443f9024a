"""Plain float64 restatement of the 8-bit paged K/V cache and the attention over it.

No reference counterpart (its caches hold the model dtype).  Numbers are e4m3 (largest 448, steps of
2^(exponent - 3) for exponents of -6 and up); an element stands for number * scale, with one power-of-two
scale per (block, KV head).  Caches here are float64 arrays of numbers [NB, Hkv, bs, D] and scales
[NB, Hkv].
"""

import numpy as np

SCALE_MIN = 2.0 ** -100


def round_e4m3(x):
    """Nearest e4m3 number, ties to even, for |x| <= 448; NaN and infinities give NaN."""
    x = np.asarray(x, np.float64)
    finite = np.where(np.isfinite(x), x, 0.0)
    _, exp = np.frexp(finite)
    step = np.exp2(np.maximum(exp - 1, -6) - 3.0)
    return np.where(np.isfinite(x), np.round(finite / step) * step, np.nan)


def scale_for(amax):
    """The least power of two s >= 2^-100 with amax <= 448 s."""
    s = SCALE_MIN
    while amax > 448.0 * s:
        s *= 2.0
    return s


def write_ref(cache, scale, rows, slots):
    """One of K / V: rows [T, Hkv, D] to flat slots [T], in place."""
    nb, hkv, bs, _ = cache.shape
    last = {}
    for t, s in enumerate(np.asarray(slots).tolist()):
        if 0 <= s < nb * bs:
            last[s] = t                       # the last token of a slot is the one written
    by_block = {}
    for s, t in last.items():
        by_block.setdefault(s // bs, []).append((s % bs, t))
    for blk, written in by_block.items():
        starts = any(off == 0 for off, _ in written)
        for h in range(hkv):
            x = np.stack([np.asarray(rows[t, h], np.float64) for _, t in written])
            mine = scale_for(float(np.max(np.abs(np.where(np.isfinite(x), x, 0.0)))))
            if starts:
                cache[blk, h] = 0.0
                new = mine
            else:
                new = max(mine, float(scale[blk, h]))
                cache[blk, h] = round_e4m3(cache[blk, h] * (scale[blk, h] / new))
            for (off, _), row in zip(written, x):
                cache[blk, h, off] = round_e4m3(row / new)
            scale[blk, h] = new


def rows_ref(cache, scale, table, count):
    """Values [count, Hkv, D] of a sequence's first positions."""
    bs = cache.shape[2]
    ids = np.asarray(table)[:-(-count // bs)] if count else np.zeros(0, np.int64)
    x = cache[ids] * scale[ids][:, :, None, None]
    return x.transpose(0, 2, 1, 3).reshape(-1, cache.shape[1], cache.shape[3])[:count]


def attend_ref(q, k, v, start, scale, causal=True, spread=False):
    """q [n, Hq, D] at positions start + i over keys j <= start + i of k, v [m, Hkv, D]: (out, bound),
    where ``bound`` [n, Hq] is max_j sum_d |q k| * scale, the size of the sums behind a score; with
    ``spread`` also [n, Hq, D] sum_j p_j |v_j - out|, p the weights."""
    n, hq, d = q.shape
    m, hkv, _ = k.shape
    out = np.empty((n, hq, v.shape[2]))
    dev = np.empty_like(out)
    bound = np.empty((n, hq))
    seen = np.arange(m)[None, :] <= np.arange(n)[:, None] + start
    if not causal:
        seen = np.ones_like(seen)
    for h in range(hq):
        kh, vh = k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]
        s = np.where(seen, q[:, h] @ kh.T * scale, -np.inf)
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        out[:, h] = p @ vh
        bound[:, h] = (np.abs(q[:, h]) @ np.abs(kh).T * scale * seen).max(1)
        if spread:
            for i in range(n):
                dev[i, h] = p[i] @ np.abs(vh - out[i, h])
    return (out, bound, dev) if spread else (out, bound)


def decode_ref(q, k8, v8, ks, vs, tables, ctx, scale):
    """q [B, Hq, D] -> (out, bound); a context of no tokens gives zeros."""
    out = np.zeros(q.shape)
    bound = np.zeros(q.shape[:2])
    for b in range(q.shape[0]):
        n = min(int(ctx[b]), tables.shape[1] * k8.shape[2])
        if n > 0:
            k, v = rows_ref(k8, ks, tables[b], n), rows_ref(v8, vs, tables[b], n)
            o, s = attend_ref(q[b:b + 1], k, v, n - 1, scale)
            out[b], bound[b] = o[0], s[0]
    return out, bound
