"""Attention over quantised caches at the ends of its ranges."""
import numpy as np
import pytest

import kvq_reference as kr
from test_gpu_kvq import BITS, attend, check_some, fill, rows

pytestmark = pytest.mark.gpu


# more rows than 65535 blocks of 32 (of 256 dimensions 16) hold, on a cache too short for long work
@pytest.mark.parametrize("n_head,hd,n_ctx,pos,M", [(65535, 2, 40, 3, 33), (2100, 2, 40, 0, 1024),
                                                   (1100, 194, 17, 0, 1024)])
@pytest.mark.parametrize("bits", BITS)
def test_the_most_rows(gpu, bits, n_head, hd, n_ctx, pos, M):
    rng = np.random.default_rng(M)
    n = min(pos + M, n_ctx)
    K, V = rows(rng, n, hd), rows(rng, n, hd)
    few = 1.5 * rng.standard_normal((8, n_head * hd), np.float32)
    q = np.tile(few, (-(-M // 8), 1))[:M]
    c = fill(gpu, bits, n_ctx, 1, hd, K, V)
    got = attend(gpu, bits, c, q, n_head, 1, hd, n_ctx, pos)
    check_some(got, q, kr.held(K, bits, hd), kr.held(V, bits, hd), n_head, 1, hd, pos, n_ctx, rng)


# one row, rows of several sizes a workgroup, several splits, and the kernel of long work
LARGE = [(4, 1, 128, 300, 200, 1), (8, 2, 64, 300, 200, 40), (32, 8, 128, 300, 10, 70), (16, 2, 256, 90, 30, 9),
         (32, 8, 128, 5000, 4990, 1), (8, 1, 96, 6000, 5900, 33), (2200, 1, 32, 520, 310, 100)]


@pytest.mark.parametrize("case", LARGE, ids=str)
@pytest.mark.parametrize("bits", BITS)
def test_the_largest_queries(gpu, bits, case):
    """Finite queries of any size, on dimensions where every key is zero: all scores are zero, so
    results are the values' means."""
    n_head, n_kv, hd, n_ctx, pos, M = case
    rng = np.random.default_rng(hd + M)
    n = pos + M
    K, V = rows(rng, n, n_kv * hd), rows(rng, n, n_kv * hd)
    K[:, 5::hd], K[:, 9::hd] = 0.0, -0.0
    q = np.zeros((M, n_head * hd), np.float32)
    sizes = np.array([1e20, 4.1e34, 4.2e34, 8.4e34, -1e37, -1.7e38, 3.4028235e38], np.float32)
    q[:, 5::hd] = np.resize(sizes, M * n_head).reshape(M, n_head)
    q[:, 9::hd] = -q[:, 5::hd]
    c = fill(gpu, bits, n_ctx, n_kv, hd, K, V)
    got = attend(gpu, bits, c, q, n_head, n_kv, hd, n_ctx, pos)
    # (the plain form of these queries: a row of zeros)
    check_some(got, np.zeros_like(q), kr.held(K, bits, hd), kr.held(V, bits, hd), n_head, n_kv, hd, pos, n_ctx, rng)


@pytest.mark.parametrize("alike", [True, False], ids=["alike", "apart"])
@pytest.mark.parametrize("case", LARGE, ids=str)
@pytest.mark.parametrize("bits", BITS)
def test_the_largest_scores(gpu, bits, case, alike):
    """Scores up to a float's range, where their own last bit is many powers of two.  Keys alike at
    every position: results are the values' means.  Keys apart, by far more than the scores may be
    off: results are the value of the largest score."""
    n_head, n_kv, hd, n_ctx, pos, M = case
    rng = np.random.default_rng(hd * M)
    n = pos + M
    K, V = rows(rng, n, n_kv * hd), rows(rng, n, n_kv * hd)
    if alike:
        K[:] = K[1]
    c = fill(gpu, bits, n_ctx, n_kv, hd, K, V)
    Kh, Vh = (np.float64(kr.held(x, bits, hd)) for x in (K, V))
    # (a score's size is at most hd max|k| max|q| / sqrt(hd))
    limit = 1e38 / (np.sqrt(hd) * np.abs(Kh).max() * 6)
    for size in (1e6, 1e8, 3e8, 1e9, 1e12, 1e20, 1e30, limit):
        q = rng.standard_normal((M, n_head * hd)).clip(-6, 6).astype(np.float32) * np.float32(size)
        got = attend(gpu, bits, c, q, n_head, n_kv, hd, n_ctx, pos)
        assert np.isfinite(got).all(), size
        if alike:
            check_some(got, np.zeros_like(q), Kh, Vh, n_head, n_kv, hd, pos, n_ctx, rng, 60)
            continue
        clear = 0
        for t, h in (divmod(int(i), n_head) for i in rng.integers(0, M * n_head, 60)):
            at, g = slice(h * hd, (h + 1) * hd), h // (n_head // n_kv)
            k, v = (x[:pos + t + 1, g * hd:(g + 1) * hd] for x in (Kh, Vh))
            s = k @ np.float64(q[t, at]) / np.sqrt(hd)
            top = (np.abs(k) @ np.abs(np.float64(q[t, at]))).max() / np.sqrt(hd)
            best = int(s.argmax())
            gap = s[best] - np.delete(s, best).max(initial=-np.inf)
            # each of two scores is off by at most (hd + 16) 2^-23 of top, as in attention_bound; 40
            # more leaves the others e^-40 together
            if gap < 2 * top * (hd + 16) * 2.0 ** -23 + 40 + np.log(n):
                continue
            clear += 1
            assert np.all(np.abs(got[t, at] - v[best]) <= 2.0 ** -20 * np.abs(v[best]) +
                          2.0 ** -31 * np.abs(v).sum(0)), (size, t, h)
        assert clear > 10, (size, clear)
