"""How far attention over a paged cache may be off by its roundings, row by row.

attention_bound (paged_reference) is what no sum of roundings can pass.  Roundings fall either way, so a row
is off by far less, and a part of the queries that went missing would hide below that bound.
Here a row's error is held, as a length over its head_dim results, to a small multiple of what
independent roundings add up to as the root of their squares, in units of 2^-24:

  scores   A query's value is held in two halves, 4 (2^-11 of the 2^-11 that the first leaves at most), or
           exactly in three bfloat16.  Products with the cache's values are exact; their sums are rounded twice
           in each matrix product of 32, of at most three parts: sqrt(6 hd / 32) of
           r = sqrt(sum_d (q_d k_d)^2 / head_dim), the root of a score's squares.  The score s is rounded
           once where it is scaled, by a factor that is rounded too, and its distance from the maximum (x in
           powers of two, the maximum 8 behind at most) once.  So a weight is off, relatively, by
           sqrt(16 + 6 hd / 32) r + |s| + |x| + 8, and the row by weight * |v - result| of that.
  weights  exp2 is off by 2, and the sum, the quotient, the parts' factors and the product by one each or two:
           12 of a product's size, root of squares over the positions, and of the result's.
  sums     Each of n / 4 matrix products of four positions rounds a sum once at most (of the waves and workgroups
           that share a row, fewer): sqrt(n / 4) of the same two sizes.

SIGMAS times the root of these three's squares: each is the most that a rounding can be, 1.7 times its
root mean square, so a row stays within five of those."""
import numpy as np

import paged_reference as pr

SIGMAS = 3.0


def rows_of(q, K, V):
    """(results, how far each row may be off) of query rows q [R][hd], in 64 bits, over K and V [n][hd]."""
    q, K, V = (np.asarray(a, np.float64) for a in (q, K, V))
    (R, hd), n = q.shape, K.shape[0]
    s = q @ K.T / np.sqrt(hd)
    x = s - s.max(1, keepdims=True)
    p = np.exp(x)
    p /= p.sum(1, keepdims=True)
    o = p @ V
    r = np.sqrt((q * q) @ (K * K).T / hd)
    score = np.sqrt(16 + 6 * hd / 32) * r + np.abs(s) - x * np.log2(np.e) + 8
    vv = (V * V).sum(1)
    away = np.maximum(vv[None, :] - 2 * (o @ V.T) + (o * o).sum(1)[:, None], 0.0)
    score2 = (p * p * score ** 2 * away).sum(1)
    size2 = (p * p) @ vv + (o * o).sum(1)
    return o, SIGMAS * 2.0 ** -24 * np.sqrt(score2 + (12 ** 2 + n / 4) * size2)


def off(got, q, kpool, vpool, table, kind, n_head, length, seq, heads=None):
    """The largest of the rows' errors over what they may be (heads: of these query heads only)."""
    n_kv, hd = kpool.shape[1], kpool.shape[3]
    G, worst = n_head // n_kv, 0.0
    got, q = (np.asarray(a).reshape(-1, n_head, hd) for a in (got, q))
    for t in range(len(length)):
        k, ok = pr.rows_of(kpool, table, seq[t], int(length[t]))
        v, _ = pr.rows_of(vpool, table, seq[t], int(length[t]))
        if not ok.any():
            continue
        for g in range(n_kv):
            mine = [h for h in range(g * G, (g + 1) * G) if heads is None or h in heads]
            if not mine:
                continue
            want, tol = rows_of(q[t, mine], pr.from_bits(k[ok, g], kind), pr.from_bits(v[ok, g], kind))
            err = np.sqrt(((got[t, mine] - want) ** 2).sum(1))
            worst = np.maximum(worst, (err / np.maximum(tol, 1e-300)).max())   # (NaN stays)
    return float(worst)


def parts_of(q, kind, drop):
    """A query row as the products take it: halves of its values times a power of two, or bfloat16 cut off, the
    last part left out or not."""
    q = np.asarray(q, np.float32)
    if kind == pr.F16:
        e = 14 - int(np.floor(np.log2(np.abs(q).max())))
        y = np.ldexp(q, e).astype(np.float32)
        hi = y.astype(np.float16)
        lo = (y - hi.astype(np.float32)).astype(np.float16)
        return np.ldexp(hi.astype(np.float64) + (0.0 if drop else lo.astype(np.float64)), -e)
    out, left = np.zeros(q.shape), q
    for i in range(2 if drop else 3):
        part = (left.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
        out += part
        left = left - part
    return out


def arithmetic(q, K, V, kind, drop=""):
    """The kernels' arithmetic in numpy, one row: a query in parts, scores and weights as floats, four waves' tiles
    of 16 positions summed in floats.  drop: "query" without its last part, "weight" with weights of 16 bits."""
    f32 = np.float32
    K, V = np.asarray(K, np.float64), np.asarray(V, np.float64)
    n, hd = K.shape
    s = (K @ parts_of(q, kind, drop == "query")).astype(f32) * f32(np.log2(np.e) / np.sqrt(hd))
    w = np.exp2((s - s.max()).astype(np.float64)).astype(f32)
    p = pr.from_bits(pr.to_bits(w, kind), kind) if drop == "weight" else w.astype(np.float64)
    m = -(-n // 64) * 64
    p, l, V = (np.concatenate([y, np.zeros((m - n, *y.shape[1:]))]) for y in (p, w.astype(np.float64), V))
    o, total = np.zeros((4, hd), f32), np.zeros(4, f32)
    for i in range(0, m, 64):
        tile = p[i:i + 64].reshape(4, 4, 4), V[i:i + 64].reshape(4, 4, 4, hd)
        for j in range(4):
            o = (o + np.einsum("wp,wpd->wd", tile[0][:, j], tile[1][:, j])).astype(f32)
        total = (total + l[i:i + 64].reshape(4, 16).sum(1)).astype(f32)
    return o.sum(0, dtype=f32) / total.sum(dtype=f32)
