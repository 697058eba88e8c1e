"""Attention over paged caches with values out of the ordinary, where one workgroup has a head's rows and
where they are divided: NaN, infinities, pages that are none, scores far apart in parts of a row."""
import numpy as np
import pytest

import paged_reference as pr
import rustfox_amd as rf
from test_gpu_paged import KINDS, NAN, Paged, attend, check
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
def test_a_nan_stays_with_those_who_see_it(gpu, kind, shape, how):
    """In one run's key, value or query: all other results and weights keep their bits."""
    n_head, n_kv, hd = shape
    G = n_head // n_kv
    for side in "kvq":
        rng = np.random.default_rng(40 + hd)
        c = cache(gpu, rng, kind, n_head, n_kv, hd, how)
        q = rng.standard_normal((3, n_head * hd)).astype(np.float32)
        had = c.weight.copy()
        clean = attend(gpu, c, q, n_head, weigh=True)
        weights = c.d_weight.numpy()
        bad, bad_w = np.zeros((3, n_head, hd), bool), np.zeros(weights.shape, bool)
        n = int(c.length[1])
        at = n - 30
        if side == "q":
            q[1, (G - 1) * hd + 5] = np.nan
            bad[1, G - 1], bad_w[1, 0, :n] = True, True
        else:
            c.pools[side == "v"][c.table[1, at // 64], 1, at % 64, 7] = NAN[kind]
            if side == "k":
                bad[1, G:2 * G], bad_w[1, 1, :n] = True, True
            else:
                bad[1, G:2 * G, 7] = True
        c.weight = had
        c.upload()
        got = attend(gpu, c, q, n_head, weigh=True).reshape(bad.shape)
        now = c.d_weight.numpy()
        assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], clean.reshape(bad.shape)[~bad])
        assert np.isnan(now[bad_w]).all() and np.array_equal(now[~bad_w], weights[~bad_w])
        if side != "q":                                      # behind the last row that is seen: not seen
            c.weight = had
            c.upload()
            short = [c.length[0], at, c.length[2]]
            check(gpu, c, q, n_head, length=short, weigh=True)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("kind", KINDS)
def test_parts_without_pages(gpu, kind, shape):
    """Runs of a division none, the first, some or the last of whose rows have a page."""
    n_head, n_kv, hd = shape
    rng = np.random.default_rng(50 + hd)
    c = cache(gpu, rng, kind, n_head, n_kv, hd, "divided")
    none = c.pools[0].shape[0]
    c.table[0, 10:60] = none
    c.table[0, 62] = 2 ** 32 - 1
    c.table[1, :30] = none + 9
    c.table[1, -1] = none
    c.table[2] = none
    c.upload()
    q = rng.standard_normal((3, n_head * hd)).astype(np.float32)
    got = check(gpu, c, q, n_head, weigh=True)
    assert (got[2] == 0).all()


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("kind", KINDS)
def test_parts_far_apart(gpu, kind, shape):
    """Keys whose size changes along the row, so that parts' greatest scores lie thousands apart, either way."""
    n_head, n_kv, hd = shape
    rng = np.random.default_rng(60 + hd)
    for gains in ((1, 300, 1), (300, 1, 0.01), (0.01, 1, 300), (100, 100, 100)):
        c = cache(gpu, rng, kind, n_head, n_kv, hd, "divided")
        for s in range(2):
            n = int(c.length[s])
            for part, gain in enumerate(gains):
                r = np.arange(n * part // 3, n * (part + 1) // 3)
                at = c.table[s, r // 64], slice(None), r % 64
                c.pools[0][at] = pr.to_bits(gain * pr.from_bits(c.pools[0][at], kind).astype(np.float32), kind)
        c.upload()
        q = (2.0 * rng.standard_normal((3, n_head * hd))).astype(np.float32)
        check(gpu, c, q, n_head, weigh=True)


@pytest.mark.parametrize("how", list(LENGTHS))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_scores_below_a_floats_range(gpu, shape, how):
    """Rows whose score is below every float have no weight; a token that sees no others gets zeros."""
    n_head, n_kv, hd = shape
    rng = np.random.default_rng(70 + hd)
    c = cache(gpu, rng, rf.BF16, n_head, n_kv, hd, how)
    q = rng.standard_normal((3, n_head * hd)).astype(np.float32)
    q[:, ::hd] = -1e30
    low = [np.arange(c.length[0]), np.arange(1, c.length[1], 2), np.zeros(0, int)]
    for s in range(3):
        r = np.arange(c.length[s])
        c.pools[0][c.table[s, r // 64], :, r % 64, 0] = 0
        r = low[s]
        c.pools[0][c.table[s, r // 64], :, r % 64, 0] = pr.to_bits(np.float32(1e30), rf.BF16)
    c.upload()
    had = c.weight.copy()
    got = attend(gpu, c, q, n_head, weigh=True)
    assert (got[0] == 0).all()
    now = c.d_weight.numpy()
    assert np.array_equal(now[0], had[0]) and np.array_equal(now[1][:, low[1]], had[1][:, low[1]])
    # the others as if those rows were not there (their first dimension takes no part)
    keep = np.arange(0, c.length[1], 2)
    for h in range(n_head):
        k, v = (pr.from_bits(p[c.table[1, keep // 64], h // (n_head // n_kv), keep % 64], rf.BF16) for p in c.pools)
        s = k[:, 1:] @ np.float64(q[1, h * hd + 1:(h + 1) * hd]) / np.sqrt(hd)
        e = np.exp(s - s.max())
        want = e @ v / e.sum()
        assert np.abs(got[1, h * hd:(h + 1) * hd] - want).max() < 2e-5


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
