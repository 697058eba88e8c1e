"""Outputs of the paged caches' calls that overlap their inputs are refused; rows that only lie between each
other's are not.  On the CPU: refused calls end before anything touches a device."""
import ctypes as C
import random

import pytest

import rustfox_amd as rf
import test_paged_args as args

FLOATS = (C.c_float * 65536)()
A = (C.addressof(FLOATS) + 15) // 16 * 16
APART = dict(store=dict(args.STORE, q=A, o=A + 4 * 4096, k=A + 4 * 8192, v=A + 4 * 16384),
             attention=dict(args.ATTN, q=A, o=A + 4 * 4096))


def overlap(*a):
    return bool(rf.probe_lib().fox_gpu_rows_overlap_probe(*a))


def test_rows_that_meet():
    rng = random.Random(1)
    met = 0
    for _ in range(4000):
        M, aw, bw = rng.randint(1, 6), rng.randint(1, 9), rng.randint(1, 9)
        sa, sb = aw + rng.choice([0, 1, 3, 9, 20]), bw + rng.choice([0, 1, 3, 9, 20])
        if rng.random() < 0.5:
            sa = sb = max(sa, sb)
        a, b = 1000 + rng.randint(0, 60), 1000 + rng.randint(0, 60)
        rows = [{x + i * s + d for i in range(M) for d in range(w)} for x, s, w in ((a, sa, aw), (b, sb, bw))]
        want = bool(rows[0] & rows[1])
        met += want
        assert overlap(4 * a, sa, aw, 4 * b, sb, bw, M) == want, (a, sa, aw, b, sb, bw, M)
    assert 400 < met < 3600


def test_long_rows():
    # a buffer of queries, keys and values side by side, with results in the place of the values
    assert not overlap(1 << 40, 3000, 1000, (1 << 40) + 8000, 3000, 1000, 1024)
    assert overlap(1 << 40, 3000, 1000, (1 << 40) + 8000, 3001, 1000, 1024)
    # (one row: strides say nothing)
    assert not overlap(1 << 40, 0, 1000, (1 << 40) + 4000, 0, 1000, 1)
    assert overlap(1 << 40, 0, 1000, (1 << 40) + 3996, 0, 1000, 1)


@pytest.mark.parametrize("name,change,why", [
    ("attention", dict(o=A), "overlaps q"), ("attention", dict(o=A + 4 * 255), "overlaps q"),
    ("attention", dict(o=A + 4, os=600, qs=300), "overlaps q"), ("attention", dict(o=A + 4, M=1), "overlaps q"),
    ("store", dict(o=A + 4), "with its stride"), ("store", dict(o=A, os=260), "with its stride"),
    ("store", dict(o=A + 4 * 255, M=1), "with its stride"), ("store", dict(o=A + 4 * 8192), "k or v"),
    ("store", dict(o=A + 4 * (16384 - 300)), "k or v"), ("store", dict(v=A + 4 * 4097), "k or v")])
def test_refused(name, change, why):
    lib = rf.gpu_lib()
    assert args.call(lib, args.CALLS[name][0], dict(APART[name], **change)) == args.ARG
    assert why in lib.fox_gpu_last_error().decode()


@pytest.mark.parametrize("name", list(APART))
def test_other_refusals_stand_by_themselves(name):
    """The bad calls of test_paged_args with their rows apart: refused for what is wrong in each."""
    lib = rf.gpu_lib()
    fn, _, bad = args.CALLS[name]
    for change, want in bad + [(dict(cache=dict(args.CACHE, **c)), want) for c, want in args.BAD_CACHES]:
        assert args.call(lib, fn, dict(APART[name], **change)) == want, change
        assert "overlap" not in lib.fox_gpu_last_error().decode(), change
