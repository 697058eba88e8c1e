"""How attention over a quantised cache is divided and launched, over the whole range of shapes that
its entry point takes: decided on the host, so tested without a GPU."""
import ctypes as C
import itertools

import pytest

import rustfox_amd as rf
import test_gpu_kvq as shapes
import test_gpu_kvq_rounding as rounding

N_CU = 256


def plan(hd, n_head, n_kv, M, n_ctx, n_cu=N_CU):
    out = (C.c_int64 * 8)()
    rf.probe_lib().fox_gpu_kvq_plan_probe(hd, n_head, n_kv, M, n_ctx, n_cu, out)
    names = "from_ few many few_blocks few_splits few_rows many_blocks many_splits".split()
    return dict(zip(names, out))


def width(hd):
    return -(-hd // 32) * 32 if hd <= 128 else 192 if hd <= 192 else 256


def check(hd, n_head, n_kv, M, n_ctx):
    p = plan(hd, n_head, n_kv, M, n_ctx)
    rows, w, what = M * (n_head // n_kv), width(hd), (hd, n_head, n_kv, M, n_ctx, p)
    assert p["few"] or p["many"], what
    # whatever the position, the kernel that takes it is launched
    for seen in {min(M, n_ctx), n_ctx, *(s for s in (p["from_"] - 1, p["from_"]) if min(M, n_ctx) <= s <= n_ctx)}:
        assert p["many" if seen >= p["from_"] else "few"], (seen, what)
    records = 0
    if p["few"]:
        per = p["few_rows"]
        assert per in ((8, 16) if w == 256 else (8, 16, 32)), what
        assert p["few_blocks"] == -(-rows // per) and 1 <= p["few_blocks"] <= 65535, what
        assert 1 <= p["few_splits"] and p["few_splits"] * 256 * n_kv * p["few_blocks"] < 1 << 40, what
        records = p["few_splits"]
    if p["many"]:
        assert w != 192 and p["many_blocks"] == -(-rows // 128) and p["many_splits"] >= 1, what
        assert n_kv * p["many_blocks"] * p["many_splits"] * 512 < 1 << 32, what
        records = max(records, p["many_splits"])
    if records > 1:
        assert rows * n_kv * records * (4 + w) * 4 < 1 << 30, what   # workspace
        merge_rows = -(-rows // 8) if records <= 16 and rows * n_kv >= 800 else rows
        assert merge_rows * 256 < 1 << 32, what


GROUPS = [1, 2, 7, 64, 128, 1100, 2100, 21000, 65535]
TOKENS = [1, 2, 8, 16, 17, 18, 32, 33, 34, 42, 43, 100, 999, 1024]
LENGTHS = [1, 17, 20, 32, 40, 41, 42, 43, 100, 1024, 4096, 131072, 1 << 30]


@pytest.mark.parametrize("hd", [2, 32, 48, 64, 80, 96, 112, 128, 130, 192, 194, 256])
def test_every_shape_has_a_launch(hd):
    """The largest groups among them: more rows than the blocks of one launch hold at 32 (16 of 256
    dimensions) a block, on caches shorter than a pass and long ones."""
    for g, M, n_ctx, n_kv in itertools.product(GROUPS, TOKENS, LENGTHS, (1, 8, 300, 32767)):
        if g * n_kv > 65535 or (width(hd) == 192 and M * g > 65535 * 32):
            continue                                         # (refused)
        check(hd, g * n_kv, n_kv, M, n_ctx)


def test_the_gpu_tests_reach_every_kernel():
    """Each width's kernels of 8, 16 and 32 rows, in one split and in several, and the one of 128
    rows, at the sizes that test_gpu_kvq_rounding runs."""
    met = set()
    for n_head, n_kv, hd, n_ctx, pos, M in rounding.MORE + shapes.ATTN_CASES + shapes.LONG_WORK + shapes.DIVISIONS:
        p, seen = plan(hd, n_head, n_kv, M, n_ctx), min(pos + M, n_ctx)
        if seen >= p["from_"]:
            met.add((width(hd), 128, p["many_splits"] > 1))
        else:
            met.add((width(hd), p["few_rows"], p["few_splits"] > 1))
    missing = [(w, per, several) for w in (32, 64, 96, 128, 192, 256) for per in (8, 16, 32, 128)
               for several in (False, True)
               if (w, per) not in ((256, 32), (192, 128)) and (w, per, several) not in met]
    assert not missing
