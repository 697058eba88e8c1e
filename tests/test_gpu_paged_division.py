"""Attention over paged caches where the rows of many tokens are divided among workgroups, or a workgroup
takes a head, by the lengths and sequences on the device; against numpy in 64 bits."""
import numpy as np
import pytest

import rustfox_amd as rf
from test_gpu_paged import Paged, check, dev
from test_paged_plan import mixed, plan

pytestmark = pytest.mark.gpu

NONE = [5, 2 ** 32 - 1]                                      # sequences that are none


def batch(name):
    """(lengths of the sequences, lengths of the tokens, their sequences)."""
    if name == "drafts":                                     # eight tokens of five sequences, some that see nothing
        rows = [4000, 3700, 3900, 4100, 3950]
        length = [n - 8 + j for n in rows for j in range(1, 9)]
        return rows, length + [0, 9, 4000, 0], [i for i in range(5) for _ in range(8)] + [4] + NONE + [0]
    if name == "mixed":                                      # a long sequence, short ones, a piece of a prompt
        length, seq = mixed(24, 9000, 100, 16, 300)
        return length[:24] + [316], length, seq
    if name == "prompt":
        return [4000], [0] + [4000 - 149 + i for i in range(149)] + [3, 17], [0] * 150 + NONE
    if name == "mixed-many":
        length, seq = mixed(50, 9000, 130, 90, 60)
        return length[:50] + [150], length + [0, 70], seq + [3, 2 ** 31]
    if name == "few-heads":                                  # fewer heads than compute units
        return [4000, 70], [70] * 30 + [4000 - 40 + i for i in range(40)], [1] * 30 + [0] * 40
    raise KeyError(name)


@pytest.mark.parametrize("name,n_head,n_kv,hd,whole", [
    ("drafts", 32, 8, 64, True), ("drafts", 8, 8, 40, True), ("drafts", 160, 4, 16, True), ("mixed", 8, 8, 64, False),
    ("mixed", 40, 8, 48, False), ("prompt", 8, 2, 128, True), ("prompt", 40, 2, 16, True), ("prompt", 2, 2, 192, True),
    ("mixed-many", 4, 2, 64, False), ("mixed-many", 34, 2, 24, False), ("few-heads", 4, 1, 128, False),
    ("few-heads", 17, 1, 32, False)], ids=str)
@pytest.mark.parametrize("kind", [rf.F16, rf.BF16])
def test_tokens_of_sequences(gpu, kind, name, n_head, n_kv, hd, whole):
    rng = np.random.default_rng(n_head + hd)
    rows, length, seq = batch(name)
    c = Paged(gpu, rng, kind, n_kv, hd, 64, rows)
    assert plan(n_head, n_kv, c.cap, len(rows), length, seq)["whole"] == whole
    q = rng.standard_normal((len(length), n_head * hd)).astype(np.float32)
    got = check(gpu, c, q, n_head, length=length, seq=seq)
    nothing = [n == 0 or s >= len(rows) for n, s in zip(length, seq)]
    assert (got[nothing] == 0).all()
    # and what lies behind the last token stays
    out = dev(gpu, np.full((len(length) + 3, n_head * hd), 9.25, np.float32))
    gpu.paged_attention(c.c, out, dev(gpu, q), n_head, len(length), dev(gpu, length, np.uint32), seq=dev(gpu, seq, np.uint32))
    assert np.array_equal(out.numpy()[:-3], got) and (out.numpy()[-3:] == 9.25).all()


def test_a_captured_call_is_divided_anew(gpu):
    """One graph over lengths that ask for a division and for none, in turn."""
    import ctypes as C
    rng = np.random.default_rng(9)
    rows, near, seq = batch("drafts")
    c = Paged(gpu, rng, rf.F16, 8, 32, 64, rows)
    far = [4100 if s == 3 else 60 for s in seq]
    assert plan(8, 8, c.cap, 5, near, seq)["whole"] and not plan(8, 8, c.cap, 5, far, seq)["whole"]
    q = rng.standard_normal((len(seq), 8 * 32)).astype(np.float32)
    want = {0: check(gpu, c, q, 8, length=near, seq=seq), 1: check(gpu, c, q, 8, length=far, seq=seq)}
    d_q, d_seq, d_len, out = dev(gpu, q), dev(gpu, seq, np.uint32), dev(gpu, near, np.uint32), dev(gpu, np.zeros_like(q))
    g, lib = C.c_void_p(), gpu.lib
    assert lib.fox_gpu_graph_begin(gpu.ctx) == 0
    gpu.paged_attention(c.c, out, d_q, 8, len(seq), d_len, seq=d_seq)
    assert lib.fox_gpu_graph_end(gpu.ctx, C.byref(g)) == 0
    for i in (0, 1, 1, 0, 1, 0):
        d_len.upload(np.array([near, far][i], np.uint32))
        out.upload(np.full_like(q, 7.0))
        assert lib.fox_gpu_graph_launch(gpu.ctx, g) == 0
        assert np.array_equal(out.numpy(), want[i])
        gpu.paged_attention(c.c, out, d_q, 8, len(seq), d_len, seq=d_seq)
        assert np.array_equal(out.numpy(), want[i])
    gpu.sync()
    lib.fox_gpu_graph_free(g)


@pytest.mark.parametrize("n,n_head,n_kv,hd", [(2, 8, 4, 64), (24, 8, 8, 40), (66, 8, 4, 64), (100, 16, 8, 16)], ids=str)
def test_caches_on_both_sides(gpu, n, n_head, n_kv, hd):
    """The longest caches of which a workgroup takes a head, and the shortest that are divided, for few and many
    heads; more sequences than a wave has lanes, some without rows."""
    rng = np.random.default_rng(n)
    caps = [cap for cap in range(32, 4096, 16)
            if plan(n_head, n_kv, cap, n, [cap] * n)["whole"] != plan(n_head, n_kv, cap + 16, n, [cap] * n)["whole"]]
    assert len(caps) == 1
    for cap in (caps[0], caps[0] + 16):
        lengths = [int(x) for x in cap * rng.random(n) ** 2]
        lengths[0], lengths[-1] = cap, 0
        c = Paged(gpu, rng, rf.BF16, n_kv, hd, 16, lengths)
        assert plan(n_head, n_kv, c.cap, n, lengths)["whole"] == (cap == caps[0])
        q = rng.standard_normal((n, n_head * hd)).astype(np.float32)
        check(gpu, c, q, n_head, weigh=True)


@pytest.mark.parametrize("n,n_head,n_kv,hd", [(65, 4, 4, 64), (96, 32, 4, 16), (300, 20, 1, 40), (256, 2, 2, 72), (257, 8, 2, 8),
                                              (1000, 3, 1, 16)], ids=str)
@pytest.mark.parametrize("kind", [rf.F16, rf.BF16])
def test_divided_past_a_waves_lanes(gpu, kind, n, n_head, n_kv, hd):
    """Many sequences' rows in equal runs, found through LDS: some sequences long, most short, some empty (the
    first and the last, neighbours), rows weighed."""
    rng = np.random.default_rng(n + hd)
    lengths = rng.integers(0, 90, n)
    lengths[rng.integers(0, n, 4)] = [3700, 3000, 64, 129]
    lengths[rng.integers(1, n, n // 8)] = 0
    lengths[[0, -1, -2]] = 0
    c = Paged(gpu, rng, kind, n_kv, hd, 128, [int(x) for x in lengths], room=3800 - int(lengths.max()))
    assert not plan(n_head, n_kv, c.cap, n, lengths)["whole"]
    q = rng.standard_normal((n, n_head * hd)).astype(np.float32)
    got = check(gpu, c, q, n_head, weigh=True)
    assert (got[lengths == 0] == 0).all()
    # (sequences given, in their order: divided alike)
    assert np.array_equal(got, check(gpu, c, q, n_head, seq=np.arange(n)))
