"""Attention over the 8-bit cache where the two f16 terms that f32 queries and weights are held in show: a case, its error bound, and what the result would be with
fewer terms.

The case.  Each token's key has one value that is not zero, so a score is one product and no sum over head_dim blurs what its rounding costs; the
scores of a row lie in [S / 2, 2 S], S = 8, so that some tokens share the weight and each brings an error of its own.

The bound, in parts of A = sum_j p_j |v_j| (u = 2^-24, f32 rows):
  score s_j: q in two terms 2^-22; hi k + lo k, both exact in f32 and added in one step 2^-23 (the tensor core may cut instead of rounding); log2(e),
    its product with the scale, and that with the page's scale u each: 9 u s_j in all, with the largest score s <= 16 and p_j off by both its
    own and the sum's error: 2 * 9 u s
  the exponents' arguments, rounded below 2^6 in both exponentials: 2 * 2^5 u ln 2, and log2 of the page's scale, 2^-22 |log2 vs| ln 2
  ex2.approx 2^-22 twice, weights in two terms 2^-22
  the products with V: 17 terms that may be cut at 2^-23 of the largest a step, 2 terms, 2 steps: 4 * 17 * 2^-23
  sums in f32, at most 16 one after another: 16 u twice
and half a step of the result's type in parts of |o|.
"""
import numpy as np

from attn_reference import HALF_STEP, LIMIT, round_e4m3

S, SCALE = 8.0, 0.125
U = 2.0 ** -24


def case(fmt, dt, n, heads, hd, seed):
    """(q [heads][hd], quantised k and v [n][hd], k's and v's scale): one kv head, one query."""
    rng = np.random.default_rng(seed)
    sign, dim = rng.choice([-1.0, 1.0], hd), rng.permutation(np.arange(max(n, hd)) % hd)[:n]
    lim = LIMIT[fmt]
    k, v = np.zeros((n, hd)), rng.uniform(-lim, lim, (n, hd))
    k[np.arange(n), dim] = sign[dim] * rng.uniform(0.6 * lim, lim, n)
    k, v = (np.rint(x) if fmt == "s8" else round_e4m3(x) for x in (k, v))
    q = (sign * (1.0 + rng.random((heads, hd)))).astype(np.float16 if dt == "f16" else np.float32)
    return q.astype(np.float64), k, v, float(np.float32(S / (lim * SCALE))), float(np.float32(1.7 / lim))


def formula(q, k, v, ks, vs):
    s = q @ (k * ks).T * SCALE
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    return p @ (v * vs), p @ np.abs(v * vs), s.max(-1)


def tolerance(o, a, s, vs, dt):
    part = 2 * 9 * U * s[:, None] + 2 ** 6 * U * np.log(2) + 2.0 ** -22 * abs(np.log2(vs)) * np.log(2) + 3 * 2.0 ** -22 + 4 * 17 * 2.0 ** -23 + 32 * U
    return HALF_STEP[dt] * np.abs(o) * 1.001 + part * a


def _terms(x, n):
    """x as the sum of n f16 terms, exact in between."""
    out, left = np.zeros_like(x), x
    for _ in range(n):
        t = left.astype(np.float16).astype(np.float64)
        out, left = out + t, left - t
    return out


def with_terms(q, k, v, ks, vs, dt, q_terms, w_terms):
    """The formula with q (rows scaled to [2^10, 2^11)) and the weights (up to 2^6) in so many f16 terms, everything else exact but the result's type."""
    up = np.exp2(10 - np.floor(np.log2(np.abs(q).max(-1, keepdims=True))))
    s = (_terms(q * up, q_terms) / up) @ (k * ks).T * SCALE * np.log2(np.e)
    w = np.exp2(s - np.ceil(s.max(-1, keepdims=True)))
    o = _terms(w * 2.0 ** 6, w_terms) / 2.0 ** 6 @ (v * vs) / w.sum(-1, keepdims=True)
    return o.astype(np.float16 if dt == "f16" else np.float32).astype(np.float64)


TOKENS = [3, 7, 20, 40]
