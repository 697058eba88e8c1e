"""Paged caches in numpy, 64 bits: the types, the tables, norm and rotation, attention of one token
a row, eviction, and how far results may be off."""
import numpy as np

F16, BF16 = 1, 30
HALF_STEP = {F16: 2.0 ** -11, BF16: 2.0 ** -8}      # of a value rounded to the type
LEAST = {F16: 2.0 ** -25, BF16: 2.0 ** -134}        # half of the least step


def to_bits(x, kind):
    """Floats rounded to the type, as 16-bit words: ties to even, halves saturate."""
    x = np.ascontiguousarray(x, np.float32)
    if kind == F16:
        return np.clip(x, -65504.0, 65504.0).astype(np.float16).view(np.uint16)
    u = x.view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + (u >> 16 & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), (u >> 16 | 0x40).astype(np.uint16), r)


def from_bits(w, kind):
    w = np.ascontiguousarray(w, np.uint16)
    if kind == F16:
        return w.view(np.float16).astype(np.float64)
    return (w.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def tables(p0, n, n_rot, base, scale=1.0, ext=0.0, beta_fast=32.0, beta_slow=1.0, orig_ctx=0.0,
           magnitude=1.0, factors=None):
    """Cosines and sines in the machine's longest floats."""
    ld = np.longdouble
    j = np.arange(n_rot // 2).astype(ld)
    f = ld(base) ** (-2 * j / n_rot)
    if factors is not None:
        f = f / factors.astype(ld)
    mix = np.zeros(n_rot // 2)
    if ext:
        lo, hi = (n_rot * np.log(orig_ctx / (2 * np.pi * b)) / (2 * np.log(base)) for b in (beta_fast, beta_slow))
        lo, hi = max(0.0, np.floor(lo)), min(n_rot - 1.0, np.ceil(hi))
        mix = ext * (1.0 - np.clip((np.arange(n_rot // 2) - lo) / max(hi - lo, 0.001), 0.0, 1.0))
    w = f * (ld(scale) * (1 - mix) + mix)
    th = (p0 + np.arange(n)).astype(ld)[:, None] * w
    return magnitude * np.cos(th), magnitude * np.sin(th), w.astype(np.float64)


def norm_rope(x, hd, w, eps, cos, sin, halves, n_rot):
    """Rows [M][heads hd] normed (w None: not), their heads' first n_rot dimensions rotated by the
    rows of cos and sin; and the sum of the products' sizes, for rounding errors."""
    x = np.asarray(x, np.float64)
    M = x.shape[0]
    x = x.reshape(M, -1, hd)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * np.float64(w)
    c, s = np.float64(cos)[:, None], np.float64(sin)[:, None]
    y, size = x.copy(), np.abs(x)
    ia, ib = (np.arange(n_rot // 2), np.arange(n_rot // 2, n_rot)) if halves else (np.arange(0, n_rot, 2),
                                                                                  np.arange(1, n_rot, 2))
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    size[..., ia], size[..., ib] = abs(a * c) + abs(b * s), abs(a * s) + abs(b * c)
    return y.reshape(M, -1), size.reshape(M, -1)


def rows_of(pool, table, seq, length):
    """[rows][kv heads][hd] words of the first `length` rows of a sequence, and which have a page.
    pool [pages][kv heads][page][hd]."""
    n_pages, n_kv, page, hd = pool.shape
    r = np.arange(min(length, table.shape[1] * page))
    pg = table[seq, r // page].astype(np.int64)
    ok = pg < n_pages
    return pool[np.where(ok, pg, 0), :, r % page], ok


def attention(q, kpool, vpool, table, kind, n_head, length, seq):
    """Results [M][n_head hd], the sizes attention_bound needs, and every row's weights by query head
    [M][n_head][rows] (lists)."""
    n_pages, n_kv, page, hd = kpool.shape
    M, G = q.shape[0], n_head // n_kv
    q = np.asarray(q, np.float64).reshape(M, n_head, hd)
    out, mag = np.zeros((M, n_head, hd)), np.zeros((M, n_head, hd))
    top, n_seen, weights = np.zeros((M, n_head)), np.zeros(M), []
    for t in range(M):
        ps = []
        if seq[t] < table.shape[0] and length[t] > 0:
            k, ok = rows_of(kpool, table, seq[t], length[t])
            v, _ = rows_of(vpool, table, seq[t], length[t])
            n_seen[t] = ok.sum()
        else:
            ok = np.zeros(0, bool)
        for h in range(n_head):
            p = np.zeros(len(ok))
            if ok.any():
                kk, vv = (from_bits(x[ok, h // G], kind) for x in (k, v))
                s = kk @ q[t, h] / np.sqrt(hd)
                e = np.exp(s - s.max())
                p[ok] = e / e.sum()
                out[t, h], mag[t, h] = p[ok] @ vv, p[ok] @ np.abs(vv)
                # (a query's value is held to 2^-38 of its head's largest, too: 2^-15 of 2^-23)
                top[t, h] = (np.abs(kk) @ (np.abs(q[t, h]) + 2.0 ** -15 * np.abs(q[t, h]).max())).max() / np.sqrt(hd)
            ps.append(p)
        weights.append(ps)
    return out.reshape(M, -1), dict(mag=mag.reshape(M, -1), top=top, n=n_seen, hd=hd), weights


def relative(sizes):
    """How far a softmax weight may be off, relatively, [M][n_head]: a score's products and sums in
    32 bits from a query held to 2^-21 of each value are off by at most (hd + 12) 2^-23 of
    the sum of their sizes, and by 4 roundings where it is scaled and shifted: twice, its own and
    the maximum's; the exponential and its scalings by 2^-20; the sum below by n + 8 roundings."""
    return 2 * sizes["top"] * (sizes["hd"] + 16) * 2.0 ** -23 + (sizes["n"][:, None] + 8) * 2.0 ** -24 + 2.0 ** -20


def attention_bound(sizes):
    """How far a result may be off: its weights (relative to the sum of weight |value|), and n + 8
    roundings of products and sums."""
    r = relative(sizes) + (sizes["n"][:, None] + 8) * 2.0 ** -24
    return sizes["mag"] * np.repeat(r, sizes["hd"], 1) + 1e-44


def evict(kpool, vpool, table, weight, position, length, keep, recent):
    """Copies of the pools and arrays after an eviction, and the new lengths."""
    kpool, vpool, weight, position = (x.copy() for x in (kpool, vpool, weight, position))
    n_pages, n_kv, page, hd = kpool.shape
    kept = []
    for s in range(table.shape[0]):
        n = min(int(length[s]), table.shape[1] * page)
        kept.append(min(n, keep))
        if n <= keep:
            continue
        for h in range(n_kv):
            w, p = weight[s, h, :n].astype(np.float64), position[s, h, :n].astype(np.int64)
            w = np.where(w > 0, w, 0.0)
            new = p > p.max() - recent
            # by (newest first, greatest weight, lowest row)
            order = sorted(range(n), key=lambda i: (not new[i], 0.0 if new[i] else -w[i], i))[:keep]
            mark = np.zeros(n, bool)
            mark[order] = True
            holes = [i for i in range(keep) if not mark[i]]
            late = [i for i in range(keep, n) if mark[i]]
            for to, fr in zip(holes, late):
                weight[s, h, to], position[s, h, to] = weight[s, h, fr], position[s, h, fr]
                a, b = table[s, to // page], table[s, fr // page]
                if a < n_pages and b < n_pages:
                    kpool[a, h, to % page] = kpool[b, h, fr % page]
                    vpool[a, h, to % page] = vpool[b, h, fr % page]
    return kpool, vpool, weight, position, np.array(kept, np.uint32)
