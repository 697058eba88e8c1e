"""Attention over paged caches with values out of the ordinary, where one workgroup has a head's rows and
where they are divided: infinities."""
import numpy as np
import pytest

import paged_reference as pr
import rustfox_amd as rf
from test_gpu_paged import KINDS, Paged, attend
from test_paged_plan import plan

pytestmark = pytest.mark.gpu

LENGTHS = {"whole": [300, 150, 40], "divided": [6000, 4100, 300]}
SHAPES = [(4, 2, 64), (8, 2, 128), (16, 2, 64), (16, 2, 192), (40, 2, 48), (6, 6, 40)]


def cache(gpu, rng, kind, n_head, n_kv, hd, how, **more):
    lengths = LENGTHS[how]
    c = Paged(gpu, rng, kind, n_kv, hd, 64, lengths, **more)
    assert plan(n_head, n_kv, c.cap, len(lengths), lengths)["whole"] == (how == "whole")
    return c


@pytest.mark.parametrize("how", list(LENGTHS))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("kind", KINDS)
def test_infinite_keys(gpu, kind, shape, how):
    """An infinite key whose score is not negative infinity gives NaN; one whose score is gives NaN or has no
    weight.  Nobody else sees either."""
    n_head, n_kv, hd = shape
    G = n_head // n_kv
    rng = np.random.default_rng(80 + hd)
    c = cache(gpu, rng, kind, n_head, n_kv, hd, how)
    q = rng.standard_normal((3, n_head * hd)).astype(np.float32)
    q[1, 7::hd] = np.abs(q[1, 7::hd]) + 0.1
    q[1, 7:G * hd:hd] *= -1
    clean = attend(gpu, c, q, n_head)
    at = int(c.length[1]) - 30
    place = c.table[1, at // 64], slice(None), at % 64
    key = c.pools[0][place].copy()
    c.pools[0][place][:, 7] = pr.to_bits(np.float32(np.inf), rf.BF16) if kind == rf.BF16 else 0x7C00
    assert np.isinf(pr.from_bits(c.pools[0][place][:, 7], kind)).all()
    c.upload()
    got = attend(gpu, c, q, n_head)
    assert np.array_equal(got[[0, 2]], clean[[0, 2]])
    assert np.isnan(got[1, G * hd:]).all()                   # (positive queries: positive infinity)
    # without the row: its scores far below the others'
    c.pools[0][place] = key
    c.pools[0][place][:] = 0
    c.pools[0][place][0, 7] = pr.to_bits(np.float32([3e4]), kind)[0]
    c.upload()
    lost = attend(gpu, c, q, n_head)
    for h in range(G):
        one, without = got[1, h * hd:(h + 1) * hd], lost[1, h * hd:(h + 1) * hd]
        assert np.isnan(one).all() or np.abs(one - without).max() < 1e-5
