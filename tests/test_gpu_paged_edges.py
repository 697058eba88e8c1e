"""Evictions at the ends of their arguments."""
import numpy as np
import pytest

import paged_reference as pr
import rustfox_amd as rf
from test_gpu_paged import Paged, dev

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cap", [96, 4800])
@pytest.mark.parametrize("kind", [rf.F16, rf.BF16])
def test_lengths_and_budgets_past_the_table(gpu, kind, cap):
    """A length past the table's rows means all of them, a budget past them cuts nothing."""
    for keep in (30, cap - 1, cap, cap + 1, 2 ** 40):
        rng = np.random.default_rng(cap)
        c = Paged(gpu, rng, kind, 2, 40, 16, [cap] * 4)
        for s in range(4):
            c.position[s] = rng.permutation(cap)
        c.upload()
        length = np.array([cap, cap + 1, 2 ** 32 - 1, 7], np.uint32)
        kept = dev(gpu, np.zeros(4, np.uint32))
        gpu.paged_evict(c.c, dev(gpu, length), kept, keep, min(keep, 11))
        k, v, w, p, m = pr.evict(*c.pools, c.table, c.weight, c.position, length, keep, min(keep, 11))
        assert np.array_equal(kept.numpy(), m) and m[3] == 7 and (m[:3] == min(cap, keep)).all()
        assert np.array_equal(c.d_position.numpy(), p) and np.array_equal(c.d_weight.numpy(), w)
        assert np.array_equal(c.k.numpy(), k) and np.array_equal(c.v.numpy(), v)
