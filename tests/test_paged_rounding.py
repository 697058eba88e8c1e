"""The row-by-row bound of paged_rounding, on the CPU: the kernels' arithmetic keeps well within it, and with a
part of the queries left out, or weights of 16 bits, it does not, at every type, head_dim and length that the
GPU tests of it use."""
import numpy as np
import pytest

import paged_reference as pr
import paged_rounding as ro
import test_gpu_paged_rounding as gpu_tests

USED = sorted({(hd, n) for _, _, hd, lengths in gpu_tests.CASES for n in lengths if n > 1})


@pytest.mark.parametrize("hd,n", USED)
@pytest.mark.parametrize("kind", [pr.F16, pr.BF16])
def test_a_missing_part_is_seen(kind, hd, n):
    rng = np.random.default_rng(n + hd)
    K, V = (pr.from_bits(pr.to_bits(x, kind), kind) for x in gpu_tests.values(rng, n, hd))
    q = gpu_tests.queries(rng, 24 if n < 2000 else 6, hd)
    want, tol = ro.rows_of(q, K, V)
    for drop in ("", "query", "weight"):
        err = [np.sqrt(((ro.arithmetic(r, K, V, kind, drop) - w) ** 2).sum()) for r, w in zip(q, want)]
        off = max(e / t for e, t in zip(err, tol))
        if not drop:
            assert off <= 0.5, off
        else:
            assert off >= 2, (drop, off)
