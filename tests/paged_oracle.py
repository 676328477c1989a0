"""The paged cache's operators in 64 bits, plain numpy, from their definitions."""
import math

import numpy as np


def rope_freqs(rot, theta, scaling, factor=1.0, trained=8192, fast=32.0, slow=1.0, low=1.0,
               high=4.0):
    i = np.arange(rot // 2)
    f = float(theta) ** (-2.0 * i / rot)
    if scaling == "linear":
        return f / factor
    if scaling == "yarn":
        def pair(turns):
            return rot * math.log(trained / (2 * math.pi * turns)) / (2 * math.log(theta))
        a, b = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rot - 1)
        r = np.clip((i - a) / (b - a if b > a else 1e-3), 0, 1)
        return f / factor * r + f * (1 - r)
    if scaling == "bands":
        keep = np.clip((trained * f / (2 * math.pi) - low) / (high - low), 0, 1)
        return f * keep + f / factor * (1 - keep)
    return f


def rope_gain(scaling, factor, gain=0.0):
    return (gain or 0.1 * math.log(factor) + 1) if scaling == "yarn" else 1.0


def rotate(x, positions, freqs, rot, pairs, gain):
    """x [rows, heads, hd] f64."""
    ang = positions.astype(np.float64)[:, None] * freqs
    c, s = gain * np.cos(ang)[:, None], gain * np.sin(ang)[:, None]
    y = x.astype(np.float64).copy()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, rot // 2),
                                                              slice(rot // 2, rot))
    xa, xb = y[..., a].copy(), y[..., b].copy()
    y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
    return y


def block_tables(cached, fresh, held, tables, free, n_free, page, n_blocks, rows, mask=None):
    """(status, tables, held, free, n_free, first_row, positions, slots) after the step."""
    n, width = tables.shape
    tables, held, free = tables.copy(), held.copy(), free.copy()
    none = np.full(rows, -1, np.int32)
    back = sum(int(h) for h, f in zip(held, fresh) if f < 0)
    bad = (cached < 0).any() or (held < 0).any() or (held > width).any() or n_free < 0 or \
        any(f >= 0 and int(c) + int(f) > 2**31 - 1 for c, f in zip(cached, fresh)) or \
        n_free + back > n_blocks
    need = [max(0, -(-(int(c) + int(f)) // page) - int(h)) if f >= 0 else 0
            for c, f, h in zip(cached, fresh, held)]
    total = int(np.maximum(fresh, 0).astype(np.int64).sum())
    status = 1 if bad else (2 * (total > rows) + 4 * any(h + d > width for h, d in zip(held, need)) +
                            8 * (sum(need) > n_free + back))
    if status:
        return status, tables, held, free, n_free, np.zeros(n + 1, np.int32), none, none.copy()
    top = n_free
    for b in range(n):
        if fresh[b] < 0:
            free[top:top + held[b]] = tables[b, :held[b]]
            top += int(held[b])
            held[b] = 0
    positions, slots, first = none, none.copy(), [0]
    for b in range(n):
        for _ in range(need[b]):
            top -= 1
            tables[b, held[b]] = free[top]
            held[b] += 1
        r = first[-1]
        for i in range(max(0, int(fresh[b]))):
            p = int(cached[b]) + i
            blk = int(tables[b, p // page])
            depth = i if mask is None else max(0, int(np.unpackbits(
                mask[r + i].view(np.uint8)).sum()) - 1)
            positions[r + i] = cached[b] + depth
            slots[r + i] = blk * page + p % page if 0 <= blk < n_blocks else -1
        first.append(r + max(0, int(fresh[b])))
    return status, tables, held, free, top, np.array(first, np.int32), positions, slots


def slot_of(tables, page, b, p):
    return int(tables[b, p // page]) * page + p % page if tables is not None else b * page + p


def sees(mask, row, i, j):
    if mask is None:
        return j <= i
    return j < 32 * mask.shape[1] and bool(int(mask[row, j // 32]) >> (j % 32) & 1)


def attention(q, k, v, tables, page, cached, first, mask=None):
    """q [rows, heads, hd]; k, v [slots, kv heads, hd].  (out, bound): the
    result and, for each row, 2^-24 max|v| (2 (hd + 4) S + len / 2 + 80): S the
    largest sum of |q k| / sqrt(hd) of a visible score, whose f32 dot product is
    (hd + 4) half steps off at most (twice that in a quotient of weights), and
    sums of up to len / 4 + 40 terms in a chain, for o and for the weights."""
    rows, heads, hd = q.shape
    out, bound = np.zeros((rows, heads, hd)), np.zeros((rows, heads, 1))
    group = heads // k.shape[1]
    for b, c in enumerate(cached):
        n = int(first[b + 1] - first[b])
        at = [slot_of(tables, page, b, p) for p in range(int(c) + n)]
        for i in range(n):
            r = int(first[b]) + i
            vis = [at[p] for p in range(int(c) + n)
                   if p < c or sees(mask, r, i, p - int(c))]
            if not vis:
                continue
            kk, vv = k[vis].astype(np.float64), v[vis].astype(np.float64)
            for h in range(heads):
                a, w = kk[:, h // group], vv[:, h // group]
                qq = q[r, h].astype(np.float64) / math.sqrt(hd)
                s = a @ qq
                e = np.exp(s - s.max())
                out[r, h] = e @ w / e.sum()
                top = float((np.abs(a) @ np.abs(qq)).max())
                bound[r, h] = 2.0**-24 * np.abs(w).max() * (2 * (hd + 4) * top +
                                                           len(at) / 2 + 80)
    return out, bound


def tree(rng, n, words, back=6):
    """Ancestor bits [n, words] of a random tree: a node's parent is one of the
    `back` before it, or the last cached position."""
    seen = np.zeros((n, 32 * words), np.uint8)
    for i in range(n):
        p = i - int(rng.integers(1, back + 1))
        if p >= 0:
            seen[i] = seen[p]
        seen[i, i] = 1
    return np.packbits(seen, axis=1, bitorder="little").view(np.uint32)


def accept(k, v, tables, page, cached, path, count):
    k, v = k.copy(), v.copy()
    for b, c in enumerate(cached):
        for i in range(int(count[b])):
            src = slot_of(tables, page, b, int(c) + int(path[b, i]))
            dst = slot_of(tables, page, b, int(c) + i)
            k[dst], v[dst] = k[src].copy(), v[src].copy()
    return k, v
