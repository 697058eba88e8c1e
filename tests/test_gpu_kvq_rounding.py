"""Attention over quantised caches, row by row against what its roundings add up to: a row whose
operands lost a half, or one bit of an upper half, is far outside (test_kvq_rounding)."""
import numpy as np
import pytest

import kvq_reference as kr
import kvq_rounding as ro
from test_gpu_kvq import ATTN_CASES, BITS, DIVISIONS, LONG_WORK, attend, fill

pytestmark = pytest.mark.gpu

# beside the cases of test_gpu_kvq, which reach every other kernel (test_kvq_plan): 32 rows of 96
# dimensions in several splits, and prompts, whose many rows meet rare roundings
MORE = [(64, 1, 96, 2439, 2399, 33), (16, 1, 80, 2445, 2308, 130), (32, 8, 128, 400, 0, 400),
        (24, 4, 256, 330, 30, 300), (16, 4, 64, 500, 100, 400)]


@pytest.mark.parametrize("case", MORE + ATTN_CASES + DIVISIONS + LONG_WORK, ids=str)
def test_rows_within_their_roundings(gpu, case):
    n_head, n_kv, hd, n_ctx, pos, M = case
    rng = np.random.default_rng(pos + 3 * M + hd)
    n = min(pos + M, n_ctx)
    K, V = (rng.standard_normal((n, n_kv * hd), np.float32) for _ in range(2))
    q = (1.5 * rng.standard_normal((M, n_head * hd), np.float32)).astype(np.float32)
    for bits in BITS:
        c = fill(gpu, bits, n_ctx, n_kv, hd, K, V)
        got = attend(gpu, bits, c, q, n_head, n_kv, hd, n_ctx, pos)
        off = ro.off(got, q, kr.held(K, bits, hd), kr.held(V, bits, hd), n_head, n_kv, hd, pos, n_ctx, rng)
        assert off <= 1, (bits, off)
