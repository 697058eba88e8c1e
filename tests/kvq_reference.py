"""The quantised cache's format, head norms, rotation and attention in numpy, 64 bits."""
import numpy as np

HALF = {4: 8, 8: 128}
CAP = {4: 224.0, 8: 120.0}
# every scale in order: m 2^-19 for the lowest exponent, then (8 + m) 2^e
SCALES = np.array([m * 2.0 ** -19 for m in range(8)] +
                  [(8 + m) * 2.0 ** (e - 19) for e in range(31) for m in range(8)])


def held(x, bits, hd):
    """Rows [n][heads hd] as a cache of that type gives them back (float32)."""
    x = np.asarray(x, np.float64)
    n, w = x.shape
    out = np.empty((n, w))
    h, scales = HALF[bits], SCALES[SCALES <= CAP[bits]]
    for base in range(0, w, hd):
        for d0 in range(0, hd, 32):
            c = slice(base + d0, base + min(d0 + 32, hd))
            g = x[:, c]
            bad = ~np.isfinite(g).all(1)
            g = np.where(bad[:, None], 0.0, g)
            need = np.maximum(np.maximum(g.max(1) / (h - 0.5), -g.min(1) / (h + 0.5)), 0.0)
            d = scales[np.minimum(np.searchsorted(scales, need), len(scales) - 1)][:, None]
            code = np.clip(np.rint(np.divide(g, d, out=np.zeros_like(g), where=d > 0)), -h, h - 1)
            out[:, c] = np.where(bad[:, None], np.nan, code * d)
    return out.astype(np.float32)


def tables(n_ctx, hd, base=10000.0):
    th = np.arange(n_ctx)[:, None] * base ** (-2.0 * np.arange(hd // 2) / hd)
    return np.cos(th).astype(np.float32), np.sin(th).astype(np.float32)


def norm_rope(x, hd, w, eps, cos, sin, halves):
    """Rows [M][heads hd] normed (w None: not) and rotated by the rows of cos and sin."""
    x = np.asarray(x, np.float64)
    M = x.shape[0]
    x = x.reshape(M, -1, hd)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * np.float64(w)
    c, s = np.float64(cos)[:, None], np.float64(sin)[:, None]
    a, b = (x[..., :hd // 2], x[..., hd // 2:]) if halves else (x[..., ::2], x[..., 1::2])
    y = np.empty_like(x)
    ya, yb = a * c - b * s, a * s + b * c
    if halves:
        y[..., :hd // 2], y[..., hd // 2:] = ya, yb
    else:
        y[..., ::2], y[..., 1::2] = ya, yb
    return y.reshape(M, -1)


def attention(q, K, V, n_head, n_kv, hd, pos, n_ctx):
    """(result, what attention_bound needs) of every token's heads, [M][n_head hd]; K, V
    [n_ctx][n_kv hd]."""
    q, K, V = (np.asarray(a, np.float64) for a in (q, K, V))
    M = q.shape[0]
    out, mag, flat = (np.empty((M, n_head * hd)) for _ in range(3))
    top = np.empty((M, n_head))
    for t in range(M):
        upto = min(pos + t + 1, n_ctx)
        for h in range(n_head):
            g = h // (n_head // n_kv)
            k, v = K[:upto, g * hd:(g + 1) * hd], V[:upto, g * hd:(g + 1) * hd]
            x = q[t, h * hd:(h + 1) * hd]
            s = k @ x / np.sqrt(hd)
            p = np.exp(s - s.max())
            p /= p.sum()
            at = slice(h * hd, (h + 1) * hd)
            out[t, at], mag[t, at], flat[t, at] = p @ v, p @ np.abs(v), np.abs(v).sum(0)
            top[t, h] = (np.abs(k) @ np.abs(x)).max() / np.sqrt(hd)
    return out, dict(mag=mag, flat=flat, top=top)


def attention_bound(sizes, n, hd):
    """How far a result may be off, element by element.  A score's products and sums in 32 bits,
    from a query held to 2^-21 of each value, are off by at most (hd + 12) 2^-23 of the sum of
    their sizes (top), and by 4 roundings of the score where it is scaled and shifted, 2^-22 of it
    twice; a weight is off by that, relatively, twice (its own and the maximum's), and by 2^-21 for
    the exponential and its split; n weights and products are summed with at most n + 8 roundings
    each, above and below the quotient: all relative to the sum of weight |value| (mag).

    The split is absolute at its end: a weight is held as two halves, the largest weight of a row as at
    least 2^7 (its maximum may lag by 2^8, 2^15 being the most), and halves end at 2^-24, so a
    weight is off by up to 2^-24 / 2^7 = 2^-31 of the largest, whatever its own size; the sum of
    the weights is at least the largest, so a result by 2^-31 of the sum of |value| (flat)."""
    mag, top = sizes["mag"], sizes["top"]
    rows = np.repeat(top, mag.shape[1] // top.shape[1], 1)
    return (mag * (2 * rows * (hd + 16) * 2.0 ** -23 + 2 * (n + 8) * 2.0 ** -24 + 2.0 ** -20) +
            sizes["flat"] * 2.0 ** -31)
