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
