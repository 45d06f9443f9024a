"""Draft verification in numpy float64, from its definitions (include/tv_draft.h): tree layout, rotation,
tree attention and the verdict.  The reference has no counterpart."""

import numpy as np


def ancestors_ref(parents, n):
    """bool [n, n]: node i sees t (itself or an ancestor); a parent that is no lower index is none."""
    seen = np.zeros((n, n), bool)
    for i in range(n):
        p = int(parents[i])
        if 0 <= p < i:
            seen[i] = seen[p]
        seen[i, i] = True
    return seen


def words_of(seen, nodes):
    """Mask words int64 [rows, ceil(nodes / 64)] of bool [rows, n], n <= nodes."""
    wide = np.zeros((seen.shape[0], -(-nodes // 64) * 64), bool)
    wide[:, :seen.shape[1]] = seen
    return np.packbits(wide, axis=1, bitorder="little").view(np.int64)


def layout_ref(parents, lens, ctx, table, block_size, num_blocks):
    b, t = parents.shape
    mask = np.zeros((b, t, -(-t // 64)), np.int64)
    positions, slots = np.zeros((b, t), np.int32), np.full((b, t), -1, np.int32)
    for i in range(b):
        n, c = min(max(int(lens[i]), 0), t), max(int(ctx[i]), 0)
        if n == 0:
            continue
        seen = ancestors_ref(parents[i], n)
        mask[i, :n] = words_of(seen, t)
        positions[i, :n] = c + seen.sum(1) - 1
        for j in range(n):
            col = (c + j) // block_size
            if col < table.shape[1] and 0 <= table[i, col] < num_blocks:
                slots[i, j] = table[i, col] * block_size + (c + j) % block_size
    return mask, positions, slots


def rope_ref(x, positions, rope, pairs):
    """x [N, H, D] float64 rotated by rope [P, R / 2, 2] at positions."""
    half = rope.shape[1]
    cs = rope.astype(np.float64)[positions]
    z = (cs[..., 0] + 1j * cs[..., 1])[:, None]
    out = x.astype(np.float64).copy()
    if pairs == "adjacent":
        turned = (x[..., 0:2 * half:2] + 1j * x[..., 1:2 * half:2]) * z
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = turned.real, turned.imag
    else:
        turned = (x[..., :half] + 1j * x[..., half:2 * half]) * z
        out[..., :half], out[..., half:2 * half] = turned.real, turned.imag
    return out


def attend_ref(q, k, v, seen, scale):
    """q [T, Hq, D] over k, v [n, Hkv, D], seen bool [T, n]; float64.  Returns (out, bound [T, Hq], dev [T, Hq, D]): bound is the
    largest sum of a seen score's absolute terms, dev sum_j p_j |v_j - out|.  Rows that see nothing are 0."""
    t, hq, d = q.shape
    hkv = k.shape[1]
    out, dev, bound = np.zeros((t, hq, d)), np.zeros((t, hq, d)), np.zeros((t, hq))
    if k.shape[0] == 0:
        return out, bound, dev
    for h in range(hq):
        kh, vh = k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]
        s = q[:, h] @ kh.T * scale
        terms = np.abs(q[:, h]) @ np.abs(kh).T * scale
        s = np.where(seen, s, -np.inf)
        top = s.max(1, keepdims=True)
        p = np.exp(s - np.where(np.isfinite(top), top, 0))
        total = p.sum(1, keepdims=True)
        p = p / np.where(total > 0, total, 1)
        out[:, h] = p @ vh
        bound[:, h] = np.where(seen, terms, 0).max(1)
        for i in range(t):
            dev[i, h] = p[i] @ np.abs(vh - out[i, h])
    return out, bound, dev


def verify_ref(logits, tokens, parents, lens, temperatures=None, uniforms=None):
    """(path, counts, next) and, for sampled rows, how near u came to a bound (relative to the whole)."""
    b, t, v = logits.shape
    path, counts = np.full((b, t), -1, np.int32), np.zeros(b, np.int32)
    following, near = np.full(b, -1, np.int32), np.full(b, np.inf)
    for i in range(b):
        n = min(max(int(lens[i]), 0), t)
        at = 0 if n else -1
        temp = 0.0 if temperatures is None or not temperatures[i] >= 2.0 ** -126 else float(temperatures[i])
        while at >= 0:
            path[i, counts[i]] = at
            counts[i] += 1
            x = logits[i, at].astype(np.float64)
            if np.isnan(x).any() or x.max() == -np.inf or (temp and x.max() == np.inf):
                break
            children = [j for j in range(at + 1, n) if parents[i, j] == at and 0 <= tokens[i, j] < v]
            nxt = -1
            if temp == 0:
                best = int(np.argmax(x))
                nxt = next((j for j in children if tokens[i, j] == best), -1)
                if nxt < 0:
                    following[i] = best
            else:
                p = np.exp((x - x.max()) / temp)
                p /= p.sum()
                u, c, met = float(uniforms[i, at]), 0.0, set()
                for j in children:
                    if tokens[i, j] in met:
                        continue
                    met.add(int(tokens[i, j]))
                    c += p[tokens[i, j]]
                    near[i] = min(near[i], abs(u - c))
                    if u < c:
                        nxt = j
                        break
                if nxt < 0:
                    p[list(met)] = 0
                    total = np.cumsum(p)
                    want = (u - c) / (1 - c) * total[-1]
                    k = min(int(np.searchsorted(total, want, side="right")), int(np.flatnonzero(p)[-1]))
                    following[i] = k
                    near[i] = min(near[i], np.abs(total - want).min())
            at = nxt
    return path, counts, following, near
