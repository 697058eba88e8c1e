"""The row-by-row bound of kvq_rounding, on the CPU: the kernels' arithmetic keeps well within it, and
with half of a product left out it does not, at every head_dim and length that the GPU tests use."""
import numpy as np
import pytest

import kvq_reference as kr
import kvq_rounding as ro
import test_gpu_kvq as shapes
import test_gpu_kvq_rounding as rounding

CASES = rounding.MORE + shapes.ATTN_CASES + shapes.LONG_WORK + shapes.DIVISIONS
USED = sorted({(hd, min(pos + M, n_ctx, 300_001)) for _, _, hd, n_ctx, pos, M in CASES})


@pytest.mark.parametrize("hd,n", USED)
def test_a_missing_half_is_seen(hd, n):
    rng = np.random.default_rng(n + hd)
    K, V = (rng.standard_normal((n, hd), np.float32) for _ in range(2))
    bits = 4 if n % 2 else 8
    K, V = kr.held(K, bits, hd), kr.held(V, bits, hd)
    q = (1.5 * rng.standard_normal((12 if n < 10_000 else 4, hd))).astype(np.float32)
    want, tol = ro.rows_of(q, K, V, np.full(len(q), n))
    for drop in ("", "query", "weight", "conversion"):
        off = max(np.sqrt(((ro.arithmetic(r, K, V, n, hd, drop) - w) ** 2).sum()) / t
                  for r, w, t in zip(q, want, tol))
        if not drop:
            assert off <= 0.5
        elif n > 1:                                          # (one position: its value, whatever its weight)
            assert off >= 4, (drop, off)
