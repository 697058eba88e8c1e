"""Head counts of the quantised-cache entry points that a sum of sizes would wrap: refused, whatever the
number of tokens."""
import pytest

import rustfox_amd as rf
from test_kvq_args import ARG, CALLS


@pytest.mark.parametrize("name", ["rope", "kvq_rope", "attention"])
@pytest.mark.parametrize("less", [1, 2, 3, 4, 1 << 16, 1 << 63])
@pytest.mark.parametrize("M", [1, 3])
def test_head_counts_past_the_largest(name, less, M):
    fn, base, _ = CALLS[name]
    change = dict(nh=(1 << 64) - less, M=M, qs=(1 << 64) - 1, os=(1 << 64) - 1)
    assert getattr(rf.gpu_lib(), fn)(*dict(base, **change).values()) == ARG, change
