"""Attention over paged caches held row by row to what independent roundings add up to (paged_rounding),
through every kernel: both types, up to four heads a kv head and more, each width, whole and ragged, one workgroup a
head and divided, with sequences given and without."""
import numpy as np
import pytest

import paged_rounding as ro
import rustfox_amd as rf
from test_gpu_paged import KINDS, Paged, attend
from test_paged_plan import plan

pytestmark = pytest.mark.gpu

SHORT, LONG = [2, 17, 200, 333], [2100, 40, 700]
WIDTHS = (64, 40, 128, 104, 192, 136, 256, 200)
CASES = [(n_head, 2, hd, lengths) for hd in WIDTHS for n_head in (2, 8, 10, 34) for lengths in (SHORT, LONG)]


def values(rng, n, hd):
    """Keys with channels of unequal size, and values."""
    return (rng.standard_normal((n, hd)) * np.exp(0.5 * rng.standard_normal(hd))).astype(np.float32), \
        rng.standard_normal((n, hd)).astype(np.float32)


def queries(rng, rows, hd):
    return (1.5 * rng.standard_normal((rows, hd))).astype(np.float32)


@pytest.mark.parametrize("n_head,n_kv,hd,lengths", CASES, ids=lambda x: str(x) if not isinstance(x, list) else str(len(x)))
@pytest.mark.parametrize("kind", KINDS)
def test_rows(gpu, kind, n_head, n_kv, hd, lengths):
    rng = np.random.default_rng(hd + n_head)
    c = Paged(gpu, rng, kind, n_kv, hd, 16, lengths)
    assert plan(n_head, n_kv, c.cap, len(lengths), lengths)["whole"] == (lengths is SHORT)
    q = queries(rng, len(lengths), n_head * hd)
    for seq in (None, np.arange(len(lengths))):
        got = attend(gpu, c, q, n_head, seq=seq)
        assert ro.off(got, q, *c.pools, c.table, kind, n_head, lengths, np.arange(len(lengths))) <= 1
