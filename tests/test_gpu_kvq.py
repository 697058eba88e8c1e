"""Quantised caches on the GPU: rows as they are held, head norms with the rotation and the
store, and attention, against numpy in 64 bits (kvq_reference)."""
import ctypes as C

import numpy as np
import pytest

import kvq_reference as kr
import rustfox_amd as rf

pytestmark = pytest.mark.gpu

BITS = [4, 8]
EPS = 1e-6


def rows(rng, n, w):
    """Rows with channels of unequal size, a zero row and a constant one among them."""
    x = rng.standard_normal((n, w)) * np.exp(0.7 * rng.standard_normal(w))
    x[n // 2] = 0.0
    x[n // 3] = 1.25
    return x.astype(np.float32)


def poisoned(gpu, bits, n_ctx, n_kv, hd):
    """A cache every byte of which is 0xFF: scales that are NaN."""
    return gpu.empty(gpu.kvq_bytes(bits, n_ctx, n_kv, hd), np.uint8).fill(0xFF)


def u32(gpu, v):
    return gpu.array(np.array([v], np.uint32))


def padded(gpu, x, stride):
    p = np.full((x.shape[0], stride), 7.5, np.float32)
    p[:, :x.shape[1]] = x
    return gpu.array(p)


def fill(gpu, bits, n_ctx, n_kv, hd, K, V):
    c = poisoned(gpu, bits, n_ctx, n_kv, hd)
    gpu.kvq_write(bits, c, n_ctx, n_kv, hd, u32(gpu, 0), K.shape[0], gpu.array(K), gpu.array(V))
    return c


def read(gpu, bits, c, n_ctx, n_kv, hd, p0, n):
    k, v = (gpu.empty((n, n_kv * hd), np.float32) for _ in range(2))
    gpu.kvq_read(bits, c, n_ctx, n_kv, hd, p0, n, k, v)
    return k.numpy(), v.numpy()


def same(a, b):
    """Equal, NaN for NaN (-0 and 0 are equal: a code of zero has no sign)."""
    return np.array_equal(a, b, equal_nan=True)


# ------------------------------------------------------------------ write, read

SHAPES = [(8, 128), (6, 48), (2, 40), (1, 256), (3, 96), (2, 10), (1, 2), (2, 130), (5, 64), (1, 32),
          (2, 192)]


@pytest.mark.parametrize("bits", BITS)
@pytest.mark.parametrize("n_kv,hd", SHAPES)
def test_rows_come_back_as_held(gpu, bits, n_kv, hd):
    """Odd runs of rows from odd positions, over a poisoned cache: exactly the format's values, and
    rows outside a run as they were."""
    rng = np.random.default_rng(hd)
    n_ctx, w = 101, n_kv * hd
    c = poisoned(gpu, bits, n_ctx, n_kv, hd)
    want_k, want_v = (np.full((n_ctx, w), np.nan, np.float32) for _ in range(2))
    for p, n in [(37, 1), (38, 2), (40, 33), (0, 5), (4, 30), (95, 6), (70, 1), (39, 1), (33, 64)]:
        K, V = rows(rng, n, w), rows(rng, n, w)
        ks, vs = (w + 3, w + 4) if n % 2 else (w + 4 - w % 4, w + 8 - w % 4)
        gpu.kvq_write(bits, c, n_ctx, n_kv, hd, u32(gpu, p), n, padded(gpu, K, ks),
                      padded(gpu, V, vs), ks, vs)
        want_k[p:p + n], want_v[p:p + n] = kr.held(K, bits, hd), kr.held(V, bits, hd)
        for p0, m in [(0, n_ctx), (p, n), (max(p - 1, 0), 2)]:
            k, v = read(gpu, bits, c, n_ctx, n_kv, hd, p0, m)
            assert same(k, want_k[p0:p0 + m]) and same(v, want_v[p0:p0 + m]), (p, n, p0, m)


@pytest.mark.parametrize("bits", BITS)
def test_whole_cache_in_one_write(gpu, bits):
    rng = np.random.default_rng(1)
    n_ctx, n_kv, hd = 1500, 4, 128
    K, V = rows(rng, n_ctx, n_kv * hd), rows(rng, n_ctx, n_kv * hd)
    c = fill(gpu, bits, n_ctx, n_kv, hd, K, V)
    k, v = read(gpu, bits, c, n_ctx, n_kv, hd, 0, n_ctx)
    assert same(k, kr.held(K, bits, hd)) and same(v, kr.held(V, bits, hd))


@pytest.mark.parametrize("bits", BITS)
def test_borders_of_the_format(gpu, bits):
    """Halves between codes, needs exactly at a scale and a bit beside it, the smallest and the
    largest scales, subnormals, signed zeros, NaN and infinities."""
    h = kr.HALF[bits]
    scales = kr.SCALES[kr.SCALES <= kr.CAP[bits]]
    out = []
    rng = np.random.default_rng(7)
    for d in scales[1:]:
        top = np.float32((h - 0.5) * d)
        low = np.float32(-(h + 0.5) * d)
        for edge in (top, np.nextafter(top, np.float32(np.inf)), np.nextafter(top, np.float32(0)),
                     low, np.nextafter(low, np.float32(-np.inf)), np.nextafter(low, np.float32(0))):
            g = (rng.integers(-h, h - 1, 32) + 0.5).astype(np.float32) * np.float32(d)
            g = np.where(rng.random(32) < 0.3, np.nextafter(g, rng.choice([-1e9, 1e9], 32).astype(np.float32)), g)
            g[rng.integers(32)] = edge
            out.append(np.clip(g, min(edge, -abs(edge) * 0.9), max(edge, abs(edge) * 0.9)))
    tiny = np.float32(2.0 ** -19)
    for g in ([1e-45] * 32, [tiny / 2] * 32, [-tiny] * 32, [0.0, -0.0] * 16, [3e38] * 32, [-3e38, 1] * 16,
              [kr.CAP[bits] * h] * 32, [np.nan] + [1.0] * 31, [1.0] * 31 + [np.inf],
              [-np.inf] + [0.0] * 31, [np.nan, np.inf] * 16):
        out.append(np.array(g, np.float32))
    n = len(out) // 4 * 4
    x = np.array(out[len(out) - n:], np.float32).reshape(n // 4, 128)
    c = fill(gpu, bits, n // 4, 1, 128, x, x[::-1].copy())
    k, v = read(gpu, bits, c, n // 4, 1, 128, 0, n // 4)
    want = kr.held(x, bits, 128)
    assert same(k, want) and same(v, want[::-1])
    fine = np.isfinite(want) & (np.abs(x) <= kr.CAP[bits] * (h - 0.5))
    assert np.abs(want - x)[fine].max() <= 0.5 * kr.CAP[bits]


@pytest.mark.parametrize("bits", BITS)
def test_rows_past_the_context_are_not_stored(gpu, bits):
    n_ctx, n_kv, hd = 50, 2, 64
    rng = np.random.default_rng(2)
    K, V = rows(rng, 8, n_kv * hd), rows(rng, 8, n_kv * hd)
    for p in (46, 49, 50, 63, 64, 2 ** 32 - 1):
        # (a block past the cache's end would be seen in the guard rows)
        guard = gpu.empty(gpu.kvq_bytes(bits, n_ctx + 64, n_kv, hd), np.uint8).fill(0xFF)
        before = guard.numpy()
        gpu.kvq_write(bits, guard, n_ctx, n_kv, hd, u32(gpu, p), 8, gpu.array(K), gpu.array(V))
        after, size = guard.numpy(), gpu.kvq_bytes(bits, n_ctx, n_kv, hd)
        assert np.array_equal(before[size:], after[size:])
        k, v = read(gpu, bits, guard, n_ctx, n_kv, hd, 0, n_ctx)
        m = max(0, n_ctx - p)
        wk, wv = (np.full((n_ctx, n_kv * hd), np.nan, np.float32) for _ in range(2))
        if m:
            wk[p:], wv[p:] = kr.held(K[:m], bits, hd), kr.held(V[:m], bits, hd)
        assert same(k, wk) and same(v, wv), p


def test_read_one_side_and_strides(gpu):
    n_ctx, n_kv, hd = 40, 3, 48
    w = n_kv * hd
    rng = np.random.default_rng(3)
    K, V = rows(rng, n_ctx, w), rows(rng, n_ctx, w)
    c = fill(gpu, 8, n_ctx, n_kv, hd, K, V)
    k = gpu.array(np.full((n_ctx, w + 5), 3.0, np.float32))
    gpu.kvq_read(8, c, n_ctx, n_kv, hd, 0, n_ctx, k, None, w + 5)
    got = k.numpy()
    assert same(got[:, :w], kr.held(K, 8, hd)) and np.all(got[:, w:] == 3.0)
    gpu.kvq_read(8, c, n_ctx, n_kv, hd, 2, 30, None, k, None, w + 5)
    got = k.numpy()
    assert same(got[:30, :w], kr.held(V, 8, hd)[2:32]) and np.all(got[:, w:] == 3.0)


# ------------------------------------------------------------ norm, rotation, store

ROPE_CASES = [  # n_head, n_kv, hd, M, pos, n_ctx
    (32, 8, 128, 1, 77, 100), (6, 6, 48, 8, 29, 40), (4, 2, 40, 3, 0, 20), (4, 1, 256, 37, 11, 60),
    (3, 3, 2, 5, 3, 9), (10, 2, 80, 33, 31, 64), (2, 1, 10, 2, 5, 8), (8, 2, 96, 70, 1, 80),
    (4, 4, 64, 6, 60, 64),                                    # two tokens past the context
    (2, 2, 130, 9, 4, 32),
]


@pytest.mark.parametrize("halves", [0, 1])
@pytest.mark.parametrize("case", ROPE_CASES, ids=str)
@pytest.mark.parametrize("bits", [32, 4, 8])
def test_norm_rope_store(gpu, bits, case, halves):
    """Computed in double and rounded to a float once: within half a float's step of the 64-bit
    result; a cached key is that float as the format holds it."""
    n_head, n_kv, hd, M, pos, n_ctx = case
    rng = np.random.default_rng(hd + M)
    nq, nk = n_head * hd, n_kv * hd
    q, k, v = rows(rng, M, nq), rows(rng, M, nk), rows(rng, M, nk)
    qn, kn = ((1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2))
    cos, sin = kr.tables(n_ctx, hd)
    m = max(0, min(M, n_ctx - pos))
    # rows 16 bytes apart (wide accesses where head_dim allows them), then a float off that
    for wq, wk, place, off in [(qn, kn, False, 0), (None, kn, True, 0), (qn, None, False, 1),
                               (None, None, True, 1), (qn, kn, True, 0)]:
        dq, dk, dv = padded(gpu, q, nq + 4), padded(gpu, k, nk + 8), padded(gpu, v, nk + 4 + off)
        dqn, dkn = (gpu.array(x) if x is not None else None for x in (wq, wk))
        do = dq if place else gpu.array(np.full((M, nq + 4), 7.5, np.float32))
        dc, ds = gpu.array(cos), gpu.array(sin)
        args = (dq, dk, dv, do, n_head, n_kv, hd, M, dqn, dkn, EPS, halves, dc, ds, u32(gpu, pos))
        st = (nq + 4, nq + 4, nk + 8, nk + 4 + off)
        if bits == 32:
            kc = gpu.array(np.full((n_ctx, nk), 9.0, np.float32))
            vc = gpu.array(np.full(((n_ctx + 3) // 4, nk, 4), 9.0, np.float32))
            gpu.norm_rope_store(*args, n_ctx, kc, vc, *st)
            gk = kc.numpy()
            gv = vc.numpy().transpose(0, 2, 1).reshape(-1, nk)[:n_ctx]
        else:
            c = poisoned(gpu, bits, n_ctx, n_kv, hd)
            gpu.kvq_norm_rope_store(*args, bits, c, n_ctx, *st)
            gk, gv = read(gpu, bits, c, n_ctx, n_kv, hd, 0, n_ctx)
        got = do.numpy()
        at = slice(pos, pos + m)
        want = kr.norm_rope(q[:m], hd, wq, EPS, cos[at], sin[at], halves)
        scale = np.sqrt((want ** 2).mean()) + 1
        assert np.all(np.abs(got[:m, :nq] - want) <= 2.0 ** -24 * np.abs(want) * (1 + 1e-6) + 1e-13 * scale)
        assert np.all(got[:, nq:] == 7.5)
        if m < M:
            assert np.array_equal(got[m:, :nq], q[m:] if place else np.full((M - m, nq), 7.5, np.float32))
        assert np.array_equal(dk.numpy()[:, :nk], k) and np.array_equal(dv.numpy()[:, :nk], v)
        turned = kr.norm_rope(k[:m], hd, wk, EPS, cos[at], sin[at], halves)
        if bits == 32:
            assert np.all(np.abs(gk[at] - turned) <= 2.0 ** -24 * np.abs(turned) * (1 + 1e-6) + 1e-13 * scale)
            assert np.array_equal(gv[at], v[:m])
            assert np.all(np.delete(gk, np.arange(pos, pos + m), 0) == 9.0)
            assert np.all(np.delete(gv, np.arange(pos, pos + m), 0) == 9.0)
        else:
            assert same(gk[at], kr.held(turned.astype(np.float32), bits, hd))
            assert same(gv[at], kr.held(v[:m], bits, hd))
            assert np.isnan(np.delete(gk, np.arange(pos, pos + m), 0)).all()


def test_norm_rope_agrees_with_rope_store(gpu):
    """Without norms and with adjacent pairs it is fox_gpu_rope_store's rotation, which rounds both
    products and their sum to floats: three half steps of the pair's size, one here."""
    n_head, n_kv, hd, M, pos, n_ctx = 8, 2, 64, 5, 3, 16
    rng = np.random.default_rng(5)
    q, k, v = (rng.standard_normal((M, n * hd)).astype(np.float32) for n in (n_head, n_kv, n_kv))
    cos, sin = kr.tables(n_ctx, hd)
    dc, ds = gpu.array(cos), gpu.array(sin)
    caches = []
    for own in (0, 1):
        dq, dk, dv = gpu.array(q), gpu.array(k), gpu.array(v)
        kc = gpu.empty(n_ctx * n_kv * hd, np.float32).fill(0)
        vc = gpu.empty(n_ctx * n_kv * hd, np.float32).fill(0)
        if own:
            gpu.norm_rope_store(dq, dk, dv, dq, n_head, n_kv, hd, M, None, None, EPS,
                                rf.PAIRS_ADJACENT, dc, ds, u32(gpu, pos), n_ctx, kc, vc)
        else:
            p = u32(gpu, pos)
            assert gpu.lib.fox_gpu_rope_store(gpu.ctx, dq.ptr, n_head * hd, dk.ptr, n_kv * hd, dv.ptr,
                                              n_kv * hd, n_head, n_kv, hd, M, dc.ptr, ds.ptr, p.ptr,
                                              n_ctx, kc.ptr, vc.ptr) == 0
        caches.append((dq.numpy(), kc.numpy(), vc.numpy()))
    size = np.abs(q).max() * 2
    for a, b in zip(*caches):
        assert np.abs(a - b).max() <= 4 * 2.0 ** -24 * size
    assert np.array_equal(caches[0][2], caches[1][2])


# ------------------------------------------------------------------ attention

ATTN_CASES = [  # n_head, n_kv, hd, n_ctx, pos, M
    (32, 8, 128, 700, 650, 1), (32, 16, 128, 300, 299, 1), (6, 6, 48, 77, 33, 1),
    (4, 1, 128, 64, 0, 1),                    # a single visible row
    (4, 1, 128, 64, 31, 1), (4, 1, 128, 64, 32, 1), (4, 1, 128, 64, 63, 1),   # ends about a tile
    (8, 2, 40, 130, 100, 4), (16, 2, 256, 257, 200, 8), (12, 1, 64, 100, 90, 3),
    (3, 3, 2, 40, 20, 3), (10, 2, 80, 300, 250, 7), (24, 1, 96, 200, 150, 2),
    (40, 1, 64, 90, 60, 5),                   # 200 query rows on one kv head
    (4, 2, 130, 120, 40, 20), (8, 8, 192, 70, 0, 40),
    (32, 8, 128, 400, 0, 64), (32, 8, 128, 400, 333, 61), (4, 4, 64, 300, 17, 200),
    (8, 2, 128, 513, 1, 511), (2, 1, 32, 1100, 70, 1000),
    (16, 4, 64, 2100, 2000, 1), (32, 8, 128, 5000, 4900, 1),                   # many splits
    (32, 16, 128, 4200, 4100, 8), (8, 2, 128, 6000, 5900, 33),
    (32, 8, 128, 5000, 10, 1), (32, 8, 128, 5000, 100, 2), (8, 2, 128, 6000, 3, 33),   # short in a long cache
    (32, 2, 128, 3000, 2900, 2), (64, 2, 64, 3000, 2950, 1), (24, 2, 192, 2000, 1990, 2),  # 32 rows, several tiles a wave
    (8, 1, 128, 40000, 39990, 1), (16, 1, 96, 40000, 39990, 1), (20, 1, 64, 20000, 19990, 3),
    (8, 4, 256, 1500, 1400, 20), (16, 2, 128, 1500, 1450, 8), (64, 16, 128, 300, 30, 256),
    (4, 2, 64, 50, 47, 6),                    # tokens past the context see all of it
    (4, 2, 64, 50, 60, 2),
]


def attend(gpu, bits, c, q, n_head, n_kv, hd, n_ctx, pos, pad=0):
    M, w = q.shape
    dq = padded(gpu, q, w + pad)
    out = gpu.array(np.full((M, w + pad), 5.0, np.float32))
    gpu.kvq_attention(out, dq, bits, c, n_head, n_kv, hd, M, u32(gpu, pos), n_ctx, w + pad, w + pad)
    got = out.numpy()
    assert np.all(got[:, w:] == 5.0)
    return got[:, :w]


def check(got, q, K, V, n_head, n_kv, hd, pos, n_ctx):
    want, sizes = kr.attention(q, K, V, n_head, n_kv, hd, pos, n_ctx)
    n = min(pos + q.shape[0], n_ctx)
    off = np.abs(got - want)
    assert np.all(off <= kr.attention_bound(sizes, n, hd)), (off / kr.attention_bound(sizes, n, hd)).max()
    # roundings fall either way: over all outputs they add up as their number's root
    rel = np.linalg.norm(off) / np.linalg.norm(sizes["mag"])
    assert rel <= 2.0 ** -24 * (32 + 4 * np.sqrt(n) + 8 * np.sqrt(hd) * max(1.0, sizes["top"].max())), rel


@pytest.mark.parametrize("case", ATTN_CASES, ids=str)
@pytest.mark.parametrize("bits", BITS)
def test_attention(gpu, bits, case):
    n_head, n_kv, hd, n_ctx, pos, M = case
    rng = np.random.default_rng(pos + M)
    n = min(pos + M, n_ctx)
    K, V = rows(rng, n, n_kv * hd), rows(rng, n, n_kv * hd)
    q = (1.5 * rng.standard_normal((M, n_head * hd))).astype(np.float32)
    c = fill(gpu, bits, n_ctx, n_kv, hd, K, V)               # (rows past n stay poisoned)
    got = attend(gpu, bits, c, q, n_head, n_kv, hd, n_ctx, pos, pad=3 if M > 2 else 0)
    check(got, q, kr.held(K, bits, hd), kr.held(V, bits, hd), n_head, n_kv, hd, pos, n_ctx)


@pytest.mark.parametrize("M", [2, 6, 40, 150])
@pytest.mark.parametrize("side", ["k", "v"])
@pytest.mark.parametrize("bits", BITS)
def test_a_nan_row_reaches_only_those_who_see_it(gpu, bits, side, M):
    """A NaN in the row of token j: earlier tokens of the pass do not see it.  A key's NaN is a
    score's, so the whole output is NaN; a value's is its group's 32 columns."""
    n_head, n_kv, hd, pos, j = 8, 2, 64, 45, M // 2
    n_ctx = pos + M + 3
    rng = np.random.default_rng(M)
    K, V = rows(rng, pos + M, n_kv * hd), rows(rng, pos + M, n_kv * hd)
    (K if side == "k" else V)[pos + j, hd + 40] = np.nan     # kv head 1, its second group
    q = rng.standard_normal((M, n_head * hd)).astype(np.float32)
    c = fill(gpu, bits, n_ctx, n_kv, hd, K, V)
    got = attend(gpu, bits, c, q, n_head, n_kv, hd, n_ctx, pos)
    hit = np.zeros((M, n_head, hd), bool)
    hit[j:, n_head // 2:, 0 if side == "k" else 32:] = True
    assert np.array_equal(np.isnan(got), hit.reshape(M, -1))
    Kz, Vz = (np.nan_to_num(kr.held(x, bits, hd)) for x in (K, V))
    want, sizes = kr.attention(q, Kz, Vz, n_head, n_kv, hd, pos, n_ctx)
    seen = ~hit.reshape(M, -1)
    if side == "k":
        seen[j:, n_head // 2 * hd:] = False
    assert np.all(np.abs(got - want)[seen] <= kr.attention_bound(sizes, pos + M, hd)[seen])


@pytest.mark.parametrize("M", [1, 5, 70])
def test_scores_far_apart(gpu, M):
    """Weights from one position alone, then from all alike; queries of very different sizes; a
    query of zeros; scores far below zero."""
    n_head, n_kv, hd, n_ctx, pos = 8, 2, 128, 300, 200
    rng = np.random.default_rng(M)
    n = pos + M
    K, V = rows(rng, n, n_kv * hd), rows(rng, n, n_kv * hd)
    K[:, :hd] = np.abs(K[:, :hd])
    q = rng.standard_normal((M, n_head * hd)).astype(np.float32)
    q[:, :hd] = -np.abs(q[:, :hd]) * 40                      # every score far below zero
    q[:, hd:2 * hd] *= 300                                   # one position takes all
    q[:, 2 * hd:3 * hd] *= 1e-30
    q[:, 3 * hd:4 * hd] = 0.0
    q[:, 4 * hd:5 * hd] = 0.0
    q[:, 4 * hd] = 1e6
    c = fill(gpu, 4, n_ctx, n_kv, hd, K, V)
    got = attend(gpu, 4, c, q, n_head, n_kv, hd, n_ctx, pos)
    want, sizes = kr.attention(q, kr.held(K, 4, hd), kr.held(V, 4, hd), n_head, n_kv, hd, pos, n_ctx)
    assert np.all(np.abs(got - want) <= kr.attention_bound(sizes, n, hd))


@pytest.mark.parametrize("M", [1, 40])
def test_a_bad_query_spoils_its_own_rows_only(gpu, M):
    n_head, n_kv, hd, n_ctx, pos = 8, 2, 64, 200, 120
    rng = np.random.default_rng(9)
    K, V = rows(rng, pos + M, n_kv * hd), rows(rng, pos + M, n_kv * hd)
    q = rng.standard_normal((M, n_head * hd)).astype(np.float32)
    q[0, 3] = np.nan                                         # head 0
    q[0, 2 * hd + 5] = np.inf                                # head 2
    c = fill(gpu, 8, n_ctx, n_kv, hd, K, V)
    got = attend(gpu, 8, c, q, n_head, n_kv, hd, n_ctx, pos).reshape(M, n_head, hd)
    bad = np.zeros((M, n_head), bool)
    bad[0, 0] = bad[0, 2] = True
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()


def test_small_and_large_values(gpu):
    """Caches whose scales are the smallest ones, and the largest: the matrix core's operands are
    then subnormal halves, and near the largest half."""
    n_head, n_kv, hd, n_ctx = 4, 1, 128, 100
    rng = np.random.default_rng(4)
    for size in (2e-6, 2e-5, 3e-4, 100.0):
        for bits in BITS:
            K, V = (rng.standard_normal((n_ctx, hd)).astype(np.float32) * np.float32(size) for _ in range(2))
            q = (rng.standard_normal((1, n_head * hd)) / size).astype(np.float32)
            c = fill(gpu, bits, n_ctx, n_kv, hd, K, V)
            got = attend(gpu, bits, c, q, n_head, n_kv, hd, n_ctx, n_ctx - 1)
            check(got, q, kr.held(K, bits, hd), kr.held(V, bits, hd), n_head, n_kv, hd, n_ctx - 1, n_ctx)


LONG_WORK = [  # n_head, n_kv, hd, n_ctx, pos, M: 9e7 pairs of a row and a position (2e7 of 256 dimensions)
    (2200, 1, 32, 520, 310, 100), (2200, 1, 32, 520, 100, 100),     # past them, and below in the same cache
    (512, 1, 64, 1100, 900, 192), (1000, 1, 90, 930, 800, 101), (512, 1, 128, 1850, 1750, 100),
    (170, 1, 256, 1300, 1200, 101), (170, 1, 256, 1300, 900, 101), (90, 1, 250, 1290, 1200, 200),
    (300, 1, 48, 900, 0, 900),                                      # as many tokens as positions
    (600, 1, 64, 800, 700, 200),                                    # and tokens past them
    (256, 1, 64, 400_000, 360_000, 1), (128, 1, 256, 40_000, 39_500, 4),   # few rows, split many ways
    (256, 1, 64, 400_000, 300_000, 1), (128, 1, 256, 40_000, 30_000, 4), (256, 1, 64, 400_000, 77, 1),
    (128, 2, 128, 13000, 12000, 60), (500, 1, 96, 10700, 10640, 17), (64, 1, 32, 5700, 5450, 250),
    (1100, 1, 32, 520, 310, 100), (520, 1, 90, 930, 800, 101), (300, 1, 64, 800, 700, 200),
    (130, 1, 256, 1300, 1200, 101), (128, 1, 64, 400_000, 350_000, 1), (128, 2, 128, 9000, 8000, 60),
]


def check_some(got, q, K, V, n_head, n_kv, hd, pos, n_ctx, rng, count=150):
    """The first and last row and some between, of a pass too large for the plain one."""
    M, group = q.shape[0], n_head // n_kv
    K, V = np.float64(K), np.float64(V)
    assert np.isfinite(got).all()
    picks = [0, M * n_head - 1, *rng.integers(0, M * n_head, count)]
    for t, h in (divmod(int(i), n_head) for i in picks):
        at, kv = slice(h * hd, (h + 1) * hd), slice(h // group * hd, (h // group + 1) * hd)
        want, sizes = kr.attention(q[t:t + 1, at], K[:, kv], V[:, kv], 1, 1, hd, min(pos + t, n_ctx - 1), n_ctx)
        off, bound = np.abs(got[t:t + 1, at] - want), kr.attention_bound(sizes, min(pos + t + 1, n_ctx), hd)
        assert np.all(off <= bound), (t, h, (off / bound).max())


@pytest.mark.parametrize("case", LONG_WORK, ids=str)
@pytest.mark.parametrize("bits", BITS)
def test_long_work(gpu, bits, case):
    n_head, n_kv, hd, n_ctx, pos, M = case
    rng = np.random.default_rng(pos + M)
    n = min(pos + M, n_ctx)
    K, V = (rng.standard_normal((n, n_kv * hd), np.float32) for _ in range(2))
    q = (1.5 * rng.standard_normal((M, n_head * hd), np.float32)).astype(np.float32)
    c = fill(gpu, bits, n_ctx, n_kv, hd, K, V)               # (rows past n stay poisoned)
    got = attend(gpu, bits, c, q, n_head, n_kv, hd, n_ctx, pos, pad=3 if M % 2 else 0)
    check_some(got, q, kr.held(K, bits, hd), kr.held(V, bits, hd), n_head, n_kv, hd, pos, n_ctx, rng,
               150 if n < 20000 else 20)


DIVISIONS = [  # n_head, n_kv, hd, n_ctx, pos, M: 8, 16 or 32 rows of a workgroup, or 128, in one or several splits, by width
    (1, 1, 24, 776, 775, 1), (66, 2, 24, 74, 11, 33), (5, 1, 24, 828, 766, 61), (64, 1, 24, 1956, 1909, 17),
    (64, 1, 32, 2671, 2420, 250), (64, 1, 48, 54, 14, 33), (64, 1, 64, 180, 30, 150), (2, 1, 80, 390, 355, 5),
    (128, 2, 80, 50, 26, 17), (500, 1, 80, 1603, 1599, 3), (500, 1, 96, 5022, 5004, 17),
    (64, 1, 112, 44, 10, 33), (16, 1, 126, 1289, 1159, 130), (16, 1, 128, 350, 200, 150),
    (64, 1, 128, 250, 100, 150), (64, 1, 150, 50, 10, 33), (16, 1, 160, 392, 359, 33),
    (128, 2, 192, 43, 10, 33), (8, 1, 150, 2337, 2177, 130), (1, 1, 200, 70, 39, 1), (16, 1, 256, 350, 200, 150),
    (120, 1, 200, 1036, 876, 130), (160, 1, 200, 1036, 876, 130),    (6, 2, 24, 2831, 2581, 250), (33, 1, 80, 926, 879, 17), (16, 1, 112, 2485, 2354, 130),
]


@pytest.mark.parametrize("case", DIVISIONS, ids=str)
@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("bits", BITS)
def test_rows_divided(gpu, bits, pad, case):
    n_head, n_kv, hd, n_ctx, pos, M = case
    rng = np.random.default_rng(pos + hd)
    n = pos + M
    K, V = (rng.standard_normal((n, n_kv * hd), np.float32) for _ in range(2))
    q = (1.5 * rng.standard_normal((M, n_head * hd), np.float32)).astype(np.float32)
    c = fill(gpu, bits, n_ctx, n_kv, hd, K, V)               # (rows past n stay poisoned)
    got = attend(gpu, bits, c, q, n_head, n_kv, hd, n_ctx, pos, pad=pad)
    check_some(got, q, kr.held(K, bits, hd), kr.held(V, bits, hd), n_head, n_kv, hd, pos, n_ctx, rng, 60)


@pytest.mark.parametrize("n_head,hd,pos", [(1340, 64, 300), (330, 256, 300), (640, 64, 300), (260, 256, 300), (16, 64, 100), (64, 64, 30),
                                           (16, 128, 200), (64, 128, 100), (16, 192, 100), (32, 192, 200),
                                           (16, 256, 200)])
@pytest.mark.parametrize("side", ["k", "v", "q"])
@pytest.mark.parametrize("bits", BITS)
def test_a_nan_in_long_work(gpu, bits, side, n_head, hd, pos):
    """As in the short passes: a key's NaN takes the rows that see it, a value's its group's columns
    of them, a query's or its infinity its own row."""
    M, j = 150, 90
    n = n_ctx = pos + M
    rng = np.random.default_rng(hd)
    K, V = rows(rng, n, hd), rows(rng, n, hd)
    q = rng.standard_normal((M, n_head * hd)).astype(np.float32)
    hit = np.zeros((M, n_head, hd), bool)
    if side == "q":
        q[j, 7 * hd + 3], q[j, 11 * hd] = np.nan, np.inf
        hit[j, 7] = hit[j, 11] = True
    else:
        (K if side == "k" else V)[pos + j, 40] = np.nan      # the second group
        hit[j:, :, slice(None) if side == "k" else slice(32, 64)] = True
    c = fill(gpu, bits, n_ctx, 1, hd, K, V)
    got = attend(gpu, bits, c, q, n_head, 1, hd, n_ctx, pos)
    assert np.array_equal(np.isnan(got), hit.reshape(M, -1))


def test_long_work_captured(gpu):
    """One capture serves positions on both sides of where long work begins: each replay against the
    eager call, bit for bit, and against the plain one."""
    n_head, n_kv, hd, n_ctx, M = 1100, 1, 64, 900, 100      # (from 819 positions on)
    rng = np.random.default_rng(5)
    K, V = rows(rng, n_ctx, hd), rows(rng, n_ctx, hd)
    Kh, Vh = kr.held(K, 4, hd), kr.held(V, 4, hd)
    c = fill(gpu, 4, n_ctx, n_kv, hd, K, V)
    q = rng.standard_normal((M, n_head * hd)).astype(np.float32)
    dq, pos = gpu.array(q), u32(gpu, 0)
    out, other = (gpu.empty((M, n_head * hd), np.float32) for _ in range(2))
    gpu.kvq_attention(out, dq, 4, c, n_head, n_kv, hd, M, pos, n_ctx)        # (any workspace is taken here)
    g = C.c_void_p()
    assert gpu.lib.fox_gpu_graph_begin(gpu.ctx) == 0
    gpu.kvq_attention(out, dq, 4, c, n_head, n_kv, hd, M, pos, n_ctx)
    assert gpu.lib.fox_gpu_graph_end(gpu.ctx, C.byref(g)) == 0
    for p in (790, 0, 730, 710, 720, 800, 30):
        pos.upload(np.array([p], np.uint32))
        out.fill(0xFF)
        assert gpu.lib.fox_gpu_graph_launch(gpu.ctx, g) == 0
        got = out.numpy()
        gpu.kvq_attention(other, dq, 4, c, n_head, n_kv, hd, M, pos, n_ctx)
        assert np.array_equal(other.numpy(), got)
        check_some(got, q, Kh, Vh, n_head, n_kv, hd, p, n_ctx, rng, 40)
    gpu.lib.fox_gpu_graph_free(g)


# ----------------------------------------------------------- as they are used

@pytest.mark.parametrize("bits", BITS)
def test_a_prompt_and_steps(gpu, bits):
    """A prompt, then single tokens, each stored and attended to, eagerly and as one captured graph
    replayed with other work of the context between; all against a cache kept in numpy."""
    n_head, n_kv, hd, n_ctx, steps = 8, 2, 64, 96, 7
    nq, nk = n_head * hd, n_kv * hd
    rng = np.random.default_rng(bits)
    cos, sin = kr.tables(n_ctx, hd)
    dc, ds = gpu.array(cos), gpu.array(sin)
    qn, kn = ((1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2))
    dqn, dkn = gpu.array(qn), gpu.array(kn)
    c = poisoned(gpu, bits, n_ctx, n_kv, hd)
    K, V = np.zeros((n_ctx, nk), np.float32), np.zeros((n_ctx, nk), np.float32)
    pos = u32(gpu, 0)

    def layer(M, q, k, v, out):
        gpu.kvq_norm_rope_store(q, k, v, q, n_head, n_kv, hd, M, dqn, dkn, EPS, rf.PAIRS_HALVES, dc,
                                ds, pos, bits, c, n_ctx)
        gpu.kvq_attention(out, q, bits, c, n_head, n_kv, hd, M, pos, n_ctx)

    def expect(p, q, k, v, got):
        M = q.shape[0]
        at = slice(p, p + M)
        qt = kr.norm_rope(q, hd, qn, EPS, cos[at], sin[at], True).astype(np.float32)
        K[at] = kr.held(kr.norm_rope(k, hd, kn, EPS, cos[at], sin[at], True).astype(np.float32), bits, hd)
        V[at] = kr.held(v, bits, hd)
        want, sizes = kr.attention(qt, K, V, n_head, n_kv, hd, p, n_ctx)
        assert np.all(np.abs(got - want) <= kr.attention_bound(sizes, p + M, hd)), p

    def data(M):
        return rows(rng, M, nq), rows(rng, M, nk), rows(rng, M, nk)

    M = 41
    q, k, v = data(M)
    out = gpu.empty((M, nq), np.float32)
    layer(M, gpu.array(q), gpu.array(k), gpu.array(v), out)
    expect(0, q, k, v, out.numpy())
    q, k, v = data(1)
    dq, dk, dv, do = gpu.array(q), gpu.array(k), gpu.array(v), gpu.empty((1, nq), np.float32)
    pos.upload(np.array([M], np.uint32))
    layer(1, dq, dk, dv, do)                                 # (eager: sizes the workspace)
    expect(M, q, k, v, do.numpy())
    g = C.c_void_p()
    assert gpu.lib.fox_gpu_graph_begin(gpu.ctx) == 0
    layer(1, dq, dk, dv, do)
    assert gpu.lib.fox_gpu_graph_end(gpu.ctx, C.byref(g)) == 0
    other = gpu.empty((1, nq), np.float32)
    for s in range(1, steps):
        q, k, v = data(1)
        for d, x in ((dq, q), (dk, k), (dv, v), (pos, np.array([M + s], np.uint32))):
            d.upload(x)
        assert gpu.lib.fox_gpu_graph_launch(gpu.ctx, g) == 0
        got = do.numpy()
        expect(M + s, q, k, v, got)
        # eager work between the replays: the same attention, the same bits
        gpu.kvq_attention(other, dq, bits, c, n_head, n_kv, hd, 1, pos, n_ctx)
        assert np.array_equal(other.numpy(), got)
    gpu.lib.fox_gpu_graph_free(g)


def test_a_captured_prompt_pass(gpu):
    """A pass of many tokens whose records fill the workspace, captured beside a single token's and
    replayed in turn, each against the eager call."""
    n_head, n_kv, hd, n_ctx = 8, 1, 128, 4000
    rng = np.random.default_rng(12)
    K, V = rows(rng, n_ctx, hd), rows(rng, n_ctx, hd)
    c = fill(gpu, 4, n_ctx, n_kv, hd, K, V)
    jobs = []
    for M, pos in ((20, 3900), (1, 3950)):
        dq = gpu.array(rng.standard_normal((M, n_head * hd)).astype(np.float32))
        out, dpos = gpu.empty((M, n_head * hd), np.float32), u32(gpu, pos)
        call = lambda M=M, dq=dq, out=out, dpos=dpos: gpu.kvq_attention(  # noqa: E731
            out, dq, 4, c, n_head, n_kv, hd, M, dpos, n_ctx)
        call()
        want = out.numpy()
        check(want, dq.numpy(), kr.held(K, 4, hd), kr.held(V, 4, hd), n_head, n_kv, hd, pos, n_ctx)
        g = C.c_void_p()
        assert gpu.lib.fox_gpu_graph_begin(gpu.ctx) == 0
        call()
        assert gpu.lib.fox_gpu_graph_end(gpu.ctx, C.byref(g)) == 0
        jobs.append((g, out, want, call))
    for turn in range(4):
        for g, out, want, call in jobs:
            out.fill(0xFF)
            assert gpu.lib.fox_gpu_graph_launch(gpu.ctx, g) == 0
            assert np.array_equal(out.numpy(), want)
            call()
            assert np.array_equal(out.numpy(), want)
    for g, *_ in jobs:
        gpu.lib.fox_gpu_graph_free(g)


def test_a_cache_past_four_gigabytes(gpu):
    """Offsets that need more than 32 bits: rows at both ends of a zeroed cache, whose other keys
    score 0 and whose other values add nothing."""
    n_head, n_kv, hd, n_ctx, bits = 2, 1, 256, 9_000_000, 8
    size = gpu.kvq_bytes(bits, n_ctx, n_kv, hd)
    assert size > 1 << 32
    rng = np.random.default_rng(8)
    c = gpu.empty(size, np.uint8).fill(0)
    n = 40
    K, V = (rng.standard_normal((2 * n, hd)).astype(np.float32) for _ in range(2))
    for i, p in ((0, 0), (n, n_ctx - n)):
        gpu.kvq_write(bits, c, n_ctx, n_kv, hd, u32(gpu, p), n, gpu.array(K[i:i + n]), gpu.array(V[i:i + n]))
        k, v = read(gpu, bits, c, n_ctx, n_kv, hd, p, n)
        assert same(k, kr.held(K[i:i + n], bits, hd)) and same(v, kr.held(V[i:i + n], bits, hd))
    Kh, Vh = np.float64(kr.held(K, bits, hd)), np.float64(kr.held(V, bits, hd))
    for M in (1, 20):
        q = (6 * rng.standard_normal((M, n_head * hd))).astype(np.float32)
        got = attend(gpu, bits, c, q, n_head, n_kv, hd, n_ctx, n_ctx - M)
        for t in range(M):
            for h in range(n_head):
                m = 2 * n - (M - 1 - t)
                s = Kh[:m] @ np.float64(q[t, h * hd:(h + 1) * hd]) / np.sqrt(hd)
                e = np.exp(s)
                want, mag = e @ Vh[:m], e @ np.abs(Vh[:m])
                total = e.sum() + n_ctx - M + 1 + t - m
                # 9e6 weights: each of the 512 .. 16384 running sums of a row adds at most 2^15 of them, a
                # half step each time; the scores' own error as in attention_bound
                top = (np.abs(Kh[:m]) @ np.abs(q[t, h * hd:(h + 1) * hd])).max() / np.sqrt(hd)
                rel = 2 * top * (hd + 16) * 2.0 ** -23 + 2 * 2.0 ** 15 * 2.0 ** -24 + 2.0 ** -20
                off = np.abs(got[t, h * hd:(h + 1) * hd] - want / total)
                assert np.all(off <= rel * mag / total + np.abs(Vh[:m]).sum(0) * 2.0 ** -31), (M, t, h)


def test_two_contexts_at_once(gpu):
    """Two contexts, two streams: each its own workspace."""
    n_head, n_kv, hd, n_ctx = 32, 8, 128, 2000
    rng = np.random.default_rng(6)
    jobs = []
    with rf.Gpu(0) as other:
        for g in (gpu, other):
            K, V = rows(rng, n_ctx, n_kv * hd), rows(rng, n_ctx, n_kv * hd)
            q = rng.standard_normal((1, n_head * hd)).astype(np.float32)
            c = fill(g, 4, n_ctx, n_kv, hd, K, V)
            jobs.append((g, c, g.array(q), g.empty((1, n_head * hd), np.float32), u32(g, n_ctx - 1), K, V, q))
            g.sync()
        for _ in range(20):
            for g, c, dq, out, pos, *_ in jobs:
                g.kvq_attention(out, dq, 4, c, n_head, n_kv, hd, 1, pos, n_ctx)
        for g, c, dq, out, pos, K, V, q in jobs:
            check(out.numpy(), q, kr.held(K, 4, hd), kr.held(V, 4, hd), n_head, n_kv, hd, n_ctx - 1, n_ctx)
        jobs.clear()
        del g, c, dq, out, pos
