"""How far attention over a quantised cache may be off by its roundings, row by row.

attention_bound (kvq_reference) is what no sum of roundings can pass.  Roundings fall either way, so a
row is off by far less, and a product that went missing would hide below that bound.  Here a
row's error is held, as a length over its head_dim results, to a small multiple of what
independent roundings add up to as the root of their squares, in units of 2^-24:

  scores   A query's value is rounded to a float once, 1, and held in two halves, 2 (11 bits, and 11 of
           the 2^-11 that is left at most); its products with the cache's values are exact and
           their sums rounded a few times, 2.  Position i's exponent
           x = (s - largest s) log2(e) + at most 15 is rounded once.  So a weight is off,
           relatively, by 5 r + |x| with r = sqrt(sum_d (q_d k_d)^2 / head_dim), and the row by
           weight * |v - result| of that.
  weights  exp2 is off by 2 and the weight's two halves, truncated, by at most 8 of it: with the quotient's
           roundings 12 of a product's size, root of squares over the positions, and of the
           result's, for truncation is one-sided.
  sums     Up to n / 32 tiles in four waves, eight rounded additions to each: sqrt(n / 16) of the
           same two sizes.
  ends     A weight ends at 2^-31 of the largest: 2^-7 of that weight times the root of all values'
           squares.

SIGMAS times the root of these four's squares: each is the most that a rounding can be, 1.7 times its
root mean square, so a row stays within five of those."""
import numpy as np

SIGMAS = 3.0


def rows_of(q, K, V, upto):
    """(results, how far each row may be off) of query rows q [R][hd], in 64 bits, over the first
    upto[r] positions of K and V [n][hd]."""
    q, K, V = (np.asarray(a, np.float64) for a in (q, K, V))
    R, hd = q.shape
    upto = np.asarray(upto)
    out, tol = np.empty((R, hd)), np.empty(R)
    step = max(1, 4_000_000 // K.shape[0])
    vv = (V * V).sum(1)
    for i in range(0, R, step):
        a, n = q[i:i + step], upto[i:i + step]
        most = int(n.max())
        k, v, w = K[:most], V[:most], vv[:most]
        s = a @ k.T / np.sqrt(hd)
        s[np.arange(most)[None, :] >= n[:, None]] = -np.inf
        x = s - s.max(1, keepdims=True)
        p = np.exp(x)
        p /= p.sum(1, keepdims=True)
        o = p @ v
        x = np.where(np.isfinite(x), 15 - x * np.log2(np.e), 0.0)
        r2 = (a * a) @ (k * k).T / hd
        p2 = p * p
        away = np.maximum(w[None, :] - 2 * (o @ v.T) + (o * o).sum(1)[:, None], 0.0)
        score2 = (p2 * (5 * np.sqrt(r2) + x) ** 2 * away).sum(1)
        size2 = p2 @ w + (o * o).sum(1)
        ends2 = (2.0 ** -7 * p.max(1)) ** 2 * np.cumsum(w)[n - 1]
        out[i:i + step] = o
        tol[i:i + step] = SIGMAS * 2.0 ** -24 * np.sqrt(score2 + (12 ** 2 + n / 16) * size2 + ends2)
    return out, tol


def off(got, q, K, V, n_head, n_kv, hd, pos, n_ctx, rng, most=3e8):
    """The largest of the rows' errors over what they may be; all rows where their products with
    the keys are few, else some."""
    M, G = q.shape[0], n_head // n_kv
    got, q = (np.asarray(a).reshape(M, n_kv, G, hd) for a in (got, q))
    worst = 0.0
    for g in range(n_kv):
        K1, V1 = (x[:min(pos + M, n_ctx), g * hd:(g + 1) * hd] for x in (K, V))
        R = int(max(4, min(M * G, most / n_kv / (K1.shape[0] * hd))))
        pick = np.arange(M * G) if R == M * G else np.unique([0, M * G - 1, *rng.integers(0, M * G, R)])
        t = pick // G
        want, tol = rows_of(q[t, g, pick % G], K1, V1, np.minimum(pos + t + 1, n_ctx))
        err = np.sqrt(((got[t, g, pick % G] - want) ** 2).sum(1))
        worst = np.maximum(worst, (err / np.maximum(tol, 1e-300)).max())   # (NaN stays)
    return float(worst)


def arithmetic(q, K, V, upto, hd, drop=""):
    """The kernels' arithmetic in numpy, one row: queries and weights in two halves, exponents from the
    row's maximum, tiles of 32 positions summed in floats by four waves.  drop: "query" or
    "weight" without its lower half, "conversion" with one upper half rounded the other way."""
    f32, f16 = np.float32, np.float16
    K, V = (np.asarray(x[:upto], np.float64) for x in (K, V))
    score = f32(np.log2(np.e) / np.sqrt(hd))
    top = f32(np.abs(q).max() * score)
    ex = int(np.frexp(top)[1]) - 1 if top else -100
    a = np.asarray(q, f32) * f32(score * f32(2.0 ** (14 - ex)))
    hi = a.astype(f16)
    lo = (a - hi.astype(f32)).astype(f16)
    if drop == "conversion":
        d = int(np.abs(a).argmax())
        hi[d] = np.nextafter(hi[d], f16(np.inf) if hi[d] < a[d] else f16(-np.inf))
    x = hi.astype(np.float64) + (0.0 if drop == "query" else lo.astype(np.float64))
    s = ((4 * K) @ x).astype(f32) * f32(2.0 ** (ex - 16))
    w = np.exp2((s - s.max() + f32(7)).astype(np.float64)).astype(f32)

    def truncated(y):                                        # to a half, toward zero
        h = y.astype(f16)
        past = h.astype(f32) > y
        h[past] = np.nextafter(h[past], f16(0))
        return h
    hi = truncated(w)
    lo = truncated(w - hi.astype(f32))
    p = hi.astype(np.float64) + (0.0 if drop == "weight" else lo.astype(np.float64))
    n = (upto + 127) // 128 * 128
    p, l, V = (np.concatenate([y, np.zeros((n - upto, *y.shape[1:]))]) for y in (p, w.astype(np.float64), V))
    pv = (p.reshape(-1, 1, 32) @ V.reshape(-1, 32, hd))[:, 0].astype(f32).reshape(-1, 4, hd)
    lw = l.reshape(-1, 4, 32).sum(2).astype(f32)
    o, total = np.cumsum(pv, 0, dtype=f32)[-1].sum(0), np.cumsum(lw, 0, dtype=f32)[-1].sum(0)
    return o * (f32(1) / total)
