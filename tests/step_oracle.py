"""Head norms with rotation, mixture-of-experts layers and logit rules in 64
bits, plain numpy, from their definitions; bounds in f32 half steps (H)."""
import math

import numpy as np

import paged_oracle as po

H = 2.0**-24


def head_norm(x, gain, eps):
    """x [rows, heads, hd], gain [heads, hd]."""
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gain


def norm_rope(x, gain, eps, positions, freqs, rot, pairs, rope_gain):
    """(result, bound).  The sum of squares is 14 half steps off at most (eight
    products in a chain and five or six sums), its mean and eps one each, of
    which a root leaves half, root and quotient one each: 10, with the two
    products 12 of |n|.  The rotation adds 7 of gain (|n_a| + |n_b|) and the
    angle position * 1e-15; one more for products of these."""
    n = head_norm(x, gain, eps)
    out = po.rotate(n, positions, freqs, rot, pairs, rope_gain)
    bound = 13 * H * np.abs(n)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, rot // 2),
                                                              slice(rot // 2, rot))
    both = rope_gain * (np.abs(n[..., a]) + np.abs(n[..., b]))
    far = np.maximum(positions, 0)[:, None, None] * 1e-15
    bound[..., a] = bound[..., b] = both * (20 * H + far)
    return out, bound


# ------------------------------------------------------------------ experts

def q4(rng, *shape, scale=0.05):
    """Random split Q4_0 matrices [..., out, in]: (f16 scales, quants)."""
    *lead, n = shape
    d = (rng.standard_normal((*lead, n // 32)) * scale).astype(np.float16)
    return d, rng.integers(0, 256, (*lead, n // 32, 16)).astype(np.uint8)


def weights(d, q):
    w = np.concatenate([q & 15, q >> 4], -1).astype(np.float64) - 8.0
    return (w * d.astype(np.float64)[..., None]).reshape(*q.shape[:-2], -1)


def choose(x, router, k, normalise):
    """(experts, weights) [rows, k] of rows of finite x."""
    # one product after the other, so that equal router rows score the same
    score = np.stack([(x.astype(np.float64) * r.astype(np.float64)).sum(1) for r in router], 1)
    order = np.argsort(-score, axis=1, kind="stable")[:, :k]
    e = np.exp(score - score.max(1, keepdims=True))
    p = np.take_along_axis(e, order, 1)
    return order, p / (p.sum(1, keepdims=True) if normalise else e.sum(1, keepdims=True))


def _product(x, w, dx):
    """x W^T and its bound: x is held to 22 bits (4 half steps, and 2^-35 of the
    row's largest), a block's 32 products and the blocks are added in f32."""
    y = x @ w.T
    mag = np.abs(x) @ np.abs(w).T
    small = 2.0**-35 * np.abs(x).max(1, keepdims=True) * np.abs(w).sum(1)
    return y, (x.shape[1] / 32 + 50) * H * mag + small + dx @ np.abs(w).T


def moe(x, router, gate, up, down, k, normalise, residual=None):
    """(y, bound, experts, weights); gate, up, down are (scales, quants)."""
    ids, p = choose(x, router, k, normalise)
    y, bound = np.zeros(x.shape), np.zeros(x.shape)
    wg, wu, wd = (weights(*m) for m in (gate, up, down))
    for e in set(ids.flatten().tolist()):
        row, j = np.nonzero(ids == e)
        xe = x[row].astype(np.float64)
        g, dg = _product(xe, wg[e], np.zeros(xe.shape))
        u, du = _product(xe, wu[e], np.zeros(xe.shape))
        silu = g / (1.0 + np.exp(-g))
        # silu's slope is 1.1 at most; exp, quotient and product
        z, dz = _product(silu * u, wd[e],
                         1.1 * dg * (np.abs(u) + du) + np.abs(silu) * du + 8 * H * np.abs(silu * u))
        w = p[row, j][:, None]
        np.add.at(y, row, w * z)
        np.add.at(bound, row, w * (dz + (k + 4) * H * np.abs(z)) + 2.0**-149 * np.abs(z))
    if residual is not None:
        y = y + residual
        bound = bound + H * np.abs(y)
    return y, bound, ids, p


# ------------------------------------------------------------------ logits

def logits(x, tokens=None, prompt=0, nodes=(), repeat=1.0, presence=0.0, frequency=0.0, bias=(),
           allowed=None):
    """One row under its rules: (logits, bound).  tokens: the request's, the
    first `prompt` its prompt's; nodes: tokens of the nodes that the row sees;
    bias: (token, value) in their order; allowed: truth values or None."""
    vocab = len(x)
    made, seen = np.zeros(vocab), np.zeros(vocab, bool)
    for i, t in enumerate(() if tokens is None else tokens):
        if 0 <= t < vocab:
            seen[t] = True
            made[t] += i >= prompt
    for t in nodes:
        if 0 <= t < vocab:
            seen[t] = True
            made[t] += 1
    with np.errstate(all="ignore"):
        l = x.astype(np.float64)
        bound = np.zeros(vocab)

        def step(new):  # a rounding
            nonlocal l, bound
            changed = new != l
            l = new
            bound = bound + np.where(changed & np.isfinite(l), H * np.abs(l), 0.0)
        f = float
        step(np.where(seen, np.where(l > 0, l / f(repeat), l * f(repeat)), l))
        bound = np.where(seen, bound * max(1.0, f(repeat)), bound)
        step(np.where(made > 0, l - f(frequency) * made, l))
        step(np.where(made > 0, l - f(presence), l))
        value = np.zeros(vocab)
        for t, v in bias:
            if 0 <= t < vocab:
                value[t] = v
        step(l + value)
    if allowed is not None:
        l = np.where(allowed, l, -np.inf)
    return l, bound


def check_top(l, bound, token, logprob):
    """token is the largest of l (which is bound off) and logprob its log
    softmax.  s = sum of exp(l_v - l_t): the logits' bounds, the difference's
    rounding (100 half steps for terms that count, those down to e^-100), exp's
    four, and 150 sums or products in a chain; log1p four half steps."""
    fine = ~np.isnan(l) & (l > -np.inf)
    if not fine.any():
        assert token == 0xffffffff and logprob == -np.inf, (token, logprob)
        return
    top = np.where(fine, l, -np.inf)
    assert fine[token], token
    assert top[token] >= top.max() - 2 * bound.max(), (token, top[token], top.max())
    ahead = np.flatnonzero(top[:token] == top[token])
    assert bound.max() > 0 or len(ahead) == 0, (token, ahead)
    with np.errstate(all="ignore"):
        s = np.exp(np.delete(l, token) - l[token]).sum()
    if np.isnan(s):
        assert np.isnan(logprob)
        return
    want = -math.log1p(s)
    tol = (2 * bound.max() + 254 * H) * s / (1 + s) + 4 * H * abs(want)
    assert abs(logprob - want) <= tol, (logprob, want, tol)
