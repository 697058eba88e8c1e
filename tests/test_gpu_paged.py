"""Paged caches on the GPU: tables, norm and rotation with the store into pages, attention of one
token a row and eviction, against numpy in 64 bits (paged_reference)."""
import numpy as np
import pytest

import paged_reference as pr
import rustfox_amd as rf

pytestmark = pytest.mark.gpu

KINDS = [rf.F16, rf.BF16]
NAN = {rf.F16: 0x7E01, rf.BF16: 0x7FC1}
EPS = 1e-6


def dev(gpu, x, dtype=None):
    return gpu.array(np.ascontiguousarray(x, dtype))


class From:
    """A device array from `lead` floats on."""

    def __init__(self, array, lead):
        self.array, self.ptr, self.numpy = array, array.at(lead), array.numpy


def padded(gpu, x, stride, lead=0):
    """Rows of x at a stride, from `lead` floats into the allocation on."""
    p = np.full((x.shape[0], stride), 7.5, np.float32)
    p[:, :x.shape[1]] = x
    return From(dev(gpu, np.concatenate([np.full(lead, 7.5, np.float32), p.reshape(-1)])), lead)


class Paged:
    """A cache on the host and its copy on the device: pages in no order, every place that no
    sequence's rows hold a NaN."""

    def __init__(self, gpu, rng, kind, n_kv, hd, page, lengths, room=0, spare=3, track=True, gain=1.0):
        self.gpu, self.kind, self.page, self.n_kv, self.hd = gpu, kind, page, n_kv, hd
        self.length = np.array(lengths, np.uint32)
        n, per = len(lengths), -(-(max(lengths) + room) // page) or 1
        pages = n * per + spare
        self.table = rng.permutation(pages)[:n * per].reshape(n, per).astype(np.uint32)
        self.cap = per * page
        self.pools = [np.full((pages, n_kv, page, hd), NAN[kind], np.uint16) for _ in range(2)]
        for s in range(n):
            r = np.arange(lengths[s])
            for i, p in enumerate(self.pools):
                x = rng.standard_normal((len(r), n_kv, hd)) * (np.exp(0.5 * rng.standard_normal(hd)) if i == 0 else 1.0)
                p[self.table[s, r // page], :, r % page] = pr.to_bits(x * gain, kind)
        self.weight = rng.random((n, n_kv, self.cap)).astype(np.float32) if track else None
        self.position = np.zeros((n, n_kv, self.cap), np.uint32) if track else None
        self.upload()

    def upload(self):
        g = self.gpu
        self.k, self.v = (dev(g, p) for p in self.pools)
        self.d_table, self.d_length = dev(g, self.table), dev(g, self.length)
        self.d_weight = dev(g, self.weight) if self.weight is not None else None
        self.d_position = dev(g, self.position) if self.weight is not None else None
        self.c = rf.PagedCache(self.kind, self.k, self.v, self.pools[0].shape[0], self.page, self.n_kv, self.hd,
                               self.d_table, self.table.shape[0], self.table.shape[1], self.d_weight, self.d_position)


# ------------------------------------------------------------------ tables

RAMP = dict(scale=1 / 16, ext=1.0, orig_ctx=8192.0, magnitude=1.2772588722239782)
TABLES = [(0, 100, 48, {}), (7, 1, 2, {}), (0, 33, 256, dict(base=1e6)), (131000, 300, 128, dict(base=500000.0)),
          (1000003, 65, 64, dict(base=1e6, scale=0.25)), (0, 257, 126, RAMP), (130001, 129, 128, dict(RAMP, base=5e5)),
          (50, 70, 96, dict(RAMP, ext=0.6, beta_fast=16.0, beta_slow=2.0, base=1e4)), (3, 90, 40, dict(factors=True)),
          ((1 << 30) - 5, 5, 10, {}), (9, 50, 34, dict(scale=0.0)), (11, 50, 24, dict(base=0.5))]


@pytest.mark.parametrize("p0,n,n_rot,how", TABLES, ids=str)
def test_tables(gpu, p0, n, n_rot, how):
    how = dict(how)
    base = how.pop("base", 10000.0)
    f = np.exp(np.linspace(-0.5, 3.0, n_rot // 2)).astype(np.float32) if how.pop("factors", False) else None
    cos, sin, w = pr.tables(p0, n, n_rot, base, factors=f, **how)
    for lead in (0, 1):                                  # 16-byte aligned, and not
        out = [From(dev(gpu, np.full(n * n_rot // 2 + lead + 8, 5.5, np.float32)), lead) for _ in range(2)]
        gpu.rope_tables(*out, n, n_rot, p0=p0, base=base, factors=dev(gpu, f) if f is not None else None, **how)
        mag = how.get("magnitude", 1.0)
        # a float's rounding, some roundings of the angle in double and the polynomials' ends
        turns = np.abs((p0 + np.arange(n))[:, None] * w)
        bound = mag * (8 * turns * 2.0 ** -52 + 2.0 ** -34)
        for o, want in zip(out, (cos, sin)):
            got = o.numpy()
            assert (got[:lead] == 5.5).all() and (got[lead + n * n_rot // 2:] == 5.5).all()
            err = np.abs(got[lead:lead + n * n_rot // 2].reshape(n, -1).astype(np.longdouble) - want)
            assert (err <= np.abs(want) * 2.0 ** -24 + bound).all(), float((err - bound).max())


# ------------------------------------------------------------------- store

STORES = [  # heads, kv heads, head_dim, page, n_rot, lengths before, tokens of each
    (32, 8, 128, 64, 128, [70, 3, 127], [1, 1, 1]), (8, 8, 48, 16, 48, [5, 31], [1, 9]),
    (6, 2, 40, 16, 22, [0, 15, 16], [2, 1, 3]), (4, 1, 256, 32, 64, [33], [40]), (5, 5, 8, 16, 8, [1], [1]),
    (12, 3, 96, 128, 90, [100, 7], [33, 1]), (2, 2, 192, 16, 2, [40], [17]), (9, 1, 72, 4096, 72, [9], [3]),
    (16, 4, 80, 16, 40, [16] * 9, [1] * 9), (40, 8, 128, 32, 96, [11], [300])]


@pytest.mark.parametrize("halves", [0, 1])
@pytest.mark.parametrize("case", STORES, ids=str)
@pytest.mark.parametrize("kind", KINDS)
def test_store(gpu, kind, case, halves):
    """With and without norms, aligned and not, in place and not, rows apart from positions; all
    other rows of the pools and the arrays as they were."""
    n_head, n_kv, hd, page, n_rot, before, tokens = case
    for mode in range(3):
        rng = np.random.default_rng(100 * hd + mode)
        c = Paged(gpu, rng, kind, n_kv, hd, page, before, room=max(tokens), track=mode != 1)
        M, n_table = sum(tokens), max(before) + max(tokens) + 50
        seq = np.repeat(np.arange(len(tokens)), tokens)
        row = np.concatenate([b + np.arange(t) for b, t in zip(before, tokens)]).astype(np.int64)
        order = rng.permutation(M)
        seq, row = seq[order], row[order]
        pos = row + (37 if mode == 2 else 0)
        q = (rng.standard_normal((M, n_head * hd)) * 1.5).astype(np.float32)
        k, v = (rng.standard_normal((M, n_kv * hd)).astype(np.float32) for _ in range(2))
        q[M // 2, :hd], k[M // 2, :hd] = 0.0, 0.0
        v[0, :4] = [1e30, -np.inf, np.nan, 1e-8]
        qn, kn = (1 + 0.1 * rng.standard_normal((2, hd))).astype(np.float32) if mode else (None, None)
        cos, sin = (x.astype(np.float32) for x in pr.tables(0, n_table, n_rot, 1e4)[:2])
        lead = int(mode == 1)
        qs, ks = n_head * hd + 3 * lead + 4 * (mode == 2), n_kv * hd + lead
        dq, dk, dv = (padded(gpu, x, s, lead) for x, s in ((q, qs), (k, ks), (v, ks)))
        out = dq if mode == 2 else padded(gpu, np.zeros_like(q), qs, lead)
        norms = dict(q_norm=dev(gpu, qn), k_norm=dev(gpu, kn), eps=EPS) if mode else {}
        gpu.paged_rope_store(c.c, dq, out, n_head, dk, dv, M, dev(gpu, pos, np.uint32), n_rot, halves, dev(gpu, cos),
                             dev(gpu, sin), n_table, seq=dev(gpu, seq, np.uint32),
                             row=dev(gpu, row, np.uint32) if mode == 2 else None, q_stride=qs, q_out_stride=qs,
                             k_stride=ks, v_stride=ks, **norms)
        want, size = pr.norm_rope(q, hd, qn, EPS, cos[pos], sin[pos], halves, n_rot)
        got = out.numpy()[lead:].reshape(M, qs)
        assert (got[:, n_head * hd:] == 7.5).all()
        # one rounding to float of what is computed in double
        assert (np.abs(got[:, :n_head * hd] - want) <= np.abs(want) * 2.0 ** -24 + size * 2.0 ** -46 + 1e-45).all()
        wk, sk = pr.norm_rope(k, hd, kn, EPS, cos[pos], sin[pos], halves, n_rot)
        new = [x.numpy() for x in (c.k, c.v)]
        kk = pr.from_bits(new[0][c.table[seq, row // page], :, row % page], kind).reshape(M, -1)
        # (rounded to a float on the way)
        slack = pr.HALF_STEP[kind] * np.abs(wk) * (1 + 2.0 ** -12) + sk * 2.0 ** -46 + pr.LEAST[kind]
        assert (np.abs(kk - wk) <= slack).all()
        assert np.array_equal(new[1][c.table[seq, row // page], :, row % page].reshape(M, -1) & 0x7FFF,
                              pr.to_bits(v, kind) & 0x7FFF) or np.isnan(v).any()
        gv = pr.from_bits(new[1][c.table[seq, row // page], :, row % page], kind).reshape(M, -1)
        assert np.array_equal(gv, pr.from_bits(pr.to_bits(v, kind), kind), equal_nan=True)
        for old, x in zip(c.pools, new):
            x, old = x.copy(), old.copy()
            for y in (x, old):
                y[c.table[seq, row // page], :, row % page] = 0
            assert np.array_equal(x, old)
        if c.d_weight:
            c.weight[seq, :, row], c.position[seq, :, row] = 0.0, pos[:, None]
            assert np.array_equal(c.d_weight.numpy(), c.weight) and np.array_equal(c.d_position.numpy(), c.position)


@pytest.mark.parametrize("kind", KINDS)
def test_store_leaves_out_what_has_no_place(gpu, kind):
    """Sequences and positions past the ends, rows past the table, pages that are none."""
    rng = np.random.default_rng(5)
    n_head, n_kv, hd, page = 4, 2, 64, 16
    c = Paged(gpu, rng, kind, n_kv, hd, page, [40, 40])
    c.table[1, 1] = c.pools[0].shape[0]
    c.table[1, 2] = 2 ** 32 - 1
    c.upload()
    seq = np.array([0, 2, 2 ** 32 - 1, 0, 0, 1, 1, 1, 0], np.uint32)
    pos = np.array([5, 5, 5, 60, 2 ** 32 - 1, 9, 9, 9, 9], np.uint32)
    row = np.array([7, 7, 7, 8, 9, 20, 33, 15, 48], np.uint32)
    turned = np.array([1, 0, 0, 0, 0, 1, 1, 1, 1], bool)
    stored = np.array([1, 0, 0, 0, 0, 0, 0, 1, 0], bool)
    M = len(seq)
    q = rng.standard_normal((M, n_head * hd)).astype(np.float32)
    k, v = (rng.standard_normal((M, n_kv * hd)).astype(np.float32) for _ in range(2))
    cos, sin = (x.astype(np.float32) for x in pr.tables(0, 60, hd, 1e4)[:2])
    out = dev(gpu, np.full_like(q, 3.5))
    gpu.paged_rope_store(c.c, dev(gpu, q), out, n_head, dev(gpu, k), dev(gpu, v), M, dev(gpu, pos), hd, 0,
                         dev(gpu, cos), dev(gpu, sin), 60, seq=dev(gpu, seq), row=dev(gpu, row))
    got = out.numpy()
    assert (got[~turned] == 3.5).all()
    at = pos[turned].astype(int)
    want, _ = pr.norm_rope(q[turned], hd, None, 0, cos[at], sin[at], 0, hd)
    assert np.abs(got[turned] - want).max() < 1e-5
    new_v = c.v.numpy()
    c.pools[1][c.table[seq[stored], row[stored] // page], :, row[stored] % page] = \
        pr.to_bits(v[stored], kind).reshape(-1, n_kv, hd)
    assert np.array_equal(new_v, c.pools[1])
    c.weight[seq[stored], :, row[stored]], c.position[seq[stored], :, row[stored]] = 0.0, pos[stored][:, None]
    assert np.array_equal(c.d_weight.numpy(), c.weight) and np.array_equal(c.d_position.numpy(), c.position)


# --------------------------------------------------------------- attention

def attend(gpu, c, q, n_head, length=None, seq=None, weigh=False, pad=0, lead=0):
    M, w = q.shape
    length = c.length if length is None else np.asarray(length, np.uint32)
    out = padded(gpu, np.full_like(q, 9.25), w + pad, lead)
    gpu.paged_attention(c.c, out, padded(gpu, q, w + pad, lead), n_head, M, dev(gpu, length),
                        seq=dev(gpu, seq, np.uint32) if seq is not None else None, weigh=weigh,
                        out_stride=w + pad, q_stride=w + pad)
    got = out.numpy()[lead:].reshape(M, w + pad)
    assert (got[:, w:] == 7.5).all()
    return got[:, :w]


def check(gpu, c, q, n_head, length=None, seq=None, weigh=False, pad=0, lead=0):
    before = c.weight.copy() if weigh else None
    got = attend(gpu, c, q, n_head, length, seq, weigh, pad, lead)
    length = c.length if length is None else np.asarray(length, np.uint32)
    seq = np.arange(len(length)) if seq is None else np.asarray(seq)
    want, sizes, weights = pr.attention(q, *c.pools, c.table, c.kind, n_head, length, seq)
    err = np.abs(got - want)
    assert (err <= pr.attention_bound(sizes)).all(), float((err - pr.attention_bound(sizes)).max())
    if weigh:
        G, rel, now = n_head // c.n_kv, pr.relative(sizes), c.d_weight.numpy()
        for t in range(len(length)):
            n = len(weights[t][0])
            for h in range(c.n_kv):
                p = np.array(weights[t][h * G:(h + 1) * G])
                full, bound = before[t, h].astype(np.float64), np.zeros(c.cap)
                full[:n] += p.sum(0)
                # every weight's error, then a rounding of each sum and a product's
                bound[:n] = (p * (rel[t, h * G:(h + 1) * G, None] + (G + 4) * 2.0 ** -24)).sum(0) + \
                    full[:n] * 2.0 ** -24 + 1e-44
                assert (np.abs(now[t, h] - full) <= bound).all()
        c.weight = now
    return got


ATTN = [  # heads, kv heads, head_dim, page, lengths
    (32, 8, 128, 64, [1, 63, 64, 65, 700]), (6, 6, 48, 16, [34, 1, 17]), (8, 8, 64, 32, [300]),
    (8, 2, 40, 16, [0, 5, 16]), (5, 1, 256, 16, [129, 2]), (12, 12, 8, 16, [50, 51]), (9, 3, 96, 4096, [4097, 10]),
    (16, 1, 128, 16, [260]), (17, 1, 64, 32, [90, 31]), (40, 1, 80, 16, [33]), (64, 2, 128, 64, [777]),
    (4, 4, 192, 16, [1000, 3]), (24, 2, 256, 128, [400]), (2, 2, 16, 16, [2500]), (28, 4, 120, 64, [128, 127, 129]),
    (32, 16, 128, 32, [1, 2, 3, 4, 5, 6, 7, 8, 9, 600, 1300])]


@pytest.mark.parametrize("weigh", [False, True])
@pytest.mark.parametrize("case", ATTN, ids=str)
@pytest.mark.parametrize("kind", KINDS)
def test_attention(gpu, kind, case, weigh):
    n_head, n_kv, hd, page, lengths = case
    rng = np.random.default_rng(hd + n_head)
    c = Paged(gpu, rng, kind, n_kv, hd, page, lengths)
    q = (1.5 * rng.standard_normal((len(lengths), n_head * hd))).astype(np.float32)
    check(gpu, c, q, n_head, weigh=weigh)
    check(gpu, c, q, n_head, weigh=weigh, pad=3, lead=1)


WIDE = [(n_head, hd) for n_head in (2, 8, 34) for hd in (64, 56, 128, 104, 192, 136, 256, 200)]


@pytest.mark.parametrize("case", WIDE, ids=str)
@pytest.mark.parametrize("kind", KINDS)
def test_every_kernel(gpu, kind, case):
    """Up to 4, 16 and more heads over a kv head, every width, whole and ragged: divided among workers
    and not, rows of one sequence each and of sequences given."""
    n_head, hd = case
    rng = np.random.default_rng(n_head * hd)
    for lengths, page in (([1100, 0, 63, 64, 65, 1, 2049], 32), ([40, 333, 16], 16)):
        c = Paged(gpu, rng, kind, 2, hd, page, lengths, room=100)
        q = (1.5 * rng.standard_normal((len(lengths), n_head * hd))).astype(np.float32)
        got = check(gpu, c, q, n_head, weigh=True)
        assert np.array_equal(got, check(gpu, c, q, n_head, seq=np.arange(len(lengths))))


@pytest.mark.parametrize("cap", [512, 528, 1104, 2048, 2064])
def test_short_caches(gpu, cap):
    """A workgroup a head or a run of units, on both sides of where that changes, for few and many
    items; more sequences than a wave has lanes, some without rows."""
    rng = np.random.default_rng(cap)
    for n, n_kv in ((2, 4), (66, 4)):
        lengths = [int(x) for x in rng.integers(0, cap + 1, n)]
        lengths[0], lengths[-1] = cap, 0
        c = Paged(gpu, rng, rf.BF16, n_kv, 64, 16, lengths)
        q = rng.standard_normal((n, 2 * n_kv * 64)).astype(np.float32)
        check(gpu, c, q, 2 * n_kv, weigh=True)


@pytest.mark.parametrize("case", [
    (1, 3, [64 * 85 * 3, 64 * 85 * 3 + 1, 64 * 85 * 4 - 1]), (1, 8, [64 * 32 * 2, 64 * 32 * 2 + 1, 3001]), (3, 8, None),
    (20, 8, None), (32, 8, None), (32, 8, [2300] * 32), (31, 8, [0, 2600] * 15 + [1]), (50, 8, None), (60, 8, [2500] * 60),
    (60, 10, None), (64, 4, None), (64, 4, [64 * k for k in range(64)])], ids=lambda c: "%d-%d-%s" % (c[0], c[1], c[2] and c[2][0]))
def test_runs_that_end_with_their_heads(gpu, case):
    """Work divided so that runs end with the heads or not, for fewer heads than compute units, fewer than
    twice as many, and more."""
    n, n_kv, lengths = case
    rng = np.random.default_rng(n + n_kv)
    for these in [[x] for x in lengths] if n == 1 else [lengths or [int(x) for x in rng.integers(0, 2700, n)]]:
        c = Paged(gpu, rng, rf.F16, n_kv, 8, 64, these, room=max(0, 2700 - max(these)))
        q = rng.standard_normal((n, n_kv * 8)).astype(np.float32)
        got = check(gpu, c, q, n_kv, weigh=True)
        assert np.array_equal(got, check(gpu, c, q, n_kv, seq=np.arange(n)))


@pytest.mark.parametrize("n_head,n_kv,hd", [(8, 8, 40), (12, 4, 64), (20, 2, 16)])
def test_a_prompt_on_a_long_cache(gpu, n_head, n_kv, hd):
    """More tokens than sequences, on both sides of as many heads as compute units."""
    rng = np.random.default_rng(n_head)
    c = Paged(gpu, rng, rf.BF16, n_kv, hd, 64, [4200, 2300])
    for M in (9, 130):
        seq = rng.integers(0, 3, M)                          # (sequence 2 is none)
        length = np.where(seq == 0, 4200 - M, 2300 - M) + np.arange(M)
        length[3] = 0
        q = rng.standard_normal((M, n_head * hd)).astype(np.float32)
        check(gpu, c, q, n_head, length=length, seq=seq)


def test_the_most_heads(gpu):
    """65535 heads of one kv head, and 4096 kv heads: the largest grids and tiles."""
    rng = np.random.default_rng(31)
    for n_head, n_kv, lengths in ((65535, 1, [70, 600]), (8192, 4096, [20]), (4096, 4096, [530])):
        c = Paged(gpu, rng, rf.F16, n_kv, 8, 16, lengths, track=n_kv > 1)
        q = rng.standard_normal((len(lengths), n_head * 8)).astype(np.float32)
        got = attend(gpu, c, q, n_head, weigh=n_kv > 1)
        some = np.unique(np.concatenate([[0, n_head - 1], rng.integers(0, n_head, 60)]))
        cols = (some[:, None] * 8 + np.arange(8)).reshape(-1)
        for t, n in enumerate(lengths):
            for h in some:
                g = h // (n_head // n_kv)
                pools = [p[:, g:g + 1] for p in c.pools]
                want, sizes, _ = pr.attention(q[t:t + 1, h * 8:h * 8 + 8], *pools, c.table, c.kind, 1, [n], [t])
                assert (np.abs(got[t:t + 1, h * 8:h * 8 + 8] - want) <= pr.attention_bound(sizes)).all()


def test_the_largest_pages(gpu):
    rng = np.random.default_rng(32)
    c = Paged(gpu, rng, rf.F16, 2, 64, 4096, [9000, 4096, 17])
    q = rng.standard_normal((3, 8 * 64)).astype(np.float32)
    check(gpu, c, q, 8, weigh=True)


def test_a_long_row(gpu):
    """Many splits of one sequence, beside short ones."""
    rng = np.random.default_rng(3)
    for kind, n_head, n_kv, hd, lengths in [(rf.F16, 4, 1, 128, [70001, 3]), (rf.BF16, 2, 2, 64, [1, 40000])]:
        c = Paged(gpu, rng, kind, n_kv, hd, 128, lengths)
        q = (1.5 * rng.standard_normal((2, n_head * hd))).astype(np.float32)
        check(gpu, c, q, n_head, weigh=True)


@pytest.mark.parametrize("kind", KINDS)
def test_many_sequences(gpu, kind):
    rng = np.random.default_rng(4)
    lengths = [int(x) for x in rng.integers(0, 90, 300)]
    c = Paged(gpu, rng, kind, 2, 64, 16, lengths)
    q = rng.standard_normal((300, 6 * 64)).astype(np.float32)
    check(gpu, c, q, 6, weigh=True)


@pytest.mark.parametrize("kind", KINDS)
def test_tokens_of_one_sequence(gpu, kind):
    """A prompt's tokens as rows of one call, in any order, and sequences that are none."""
    rng = np.random.default_rng(6)
    c = Paged(gpu, rng, kind, 2, 128, 16, [100, 60])
    seq = np.array([0] * 40 + [1] * 20 + [2, 2 ** 32 - 1, 0])
    length = np.concatenate([rng.permutation(100)[:40] + 1, np.arange(20) + 41, [5, 5, 0]])
    q = rng.standard_normal((len(seq), 8 * 128)).astype(np.float32)
    got = check(gpu, c, q, 8, length, seq)
    assert (got[-3:] == 0).all()


def test_many_tokens_and_rows_behind_them(gpu):
    """More tokens than a wave has lanes, of few sequences and of some that are none; what lies behind
    the last token stays."""
    rng = np.random.default_rng(33)
    c = Paged(gpu, rng, rf.BF16, 2, 64, 16, [700, 60, 1])
    seq = rng.integers(0, 5, 130).astype(np.uint32)
    seq[5] = 2 ** 32 - 1
    length = rng.integers(0, 700, 130)
    length[seq < 3] = np.minimum(length, c.length[np.minimum(seq, 2)])[seq < 3]
    q = rng.standard_normal((130, 8 * 64)).astype(np.float32)
    check(gpu, c, q, 8, length, seq)
    out = dev(gpu, np.full((140, 8 * 64), 9.25, np.float32))
    gpu.paged_attention(c.c, out, dev(gpu, q), 8, 130, dev(gpu, length, np.uint32), seq=dev(gpu, seq))
    got = out.numpy()
    assert (got[130:] == 9.25).all() and (got[:130][seq >= 3] == 0).all()
    before = c.d_weight.numpy()
    gpu.paged_attention(c.c, out, dev(gpu, q), 8, 2, dev(gpu, [0, 7], np.uint32), weigh=True)
    after = c.d_weight.numpy()
    assert np.array_equal(after[0], before[0]) and np.array_equal(after[2], before[2])
    assert np.array_equal(after[1, :, 7:], before[1, :, 7:]) and (after[1, :, :7] > before[1, :, :7]).any()


@pytest.mark.parametrize("kind", KINDS)
def test_pages_that_are_none(gpu, kind):
    """Rows without a page are hidden, whole sequences too; a length past the table's rows means all
    of them; pages shared by two sequences."""
    rng = np.random.default_rng(7)
    c = Paged(gpu, rng, kind, 2, 64, 16, [160, 160, 160, 160])
    c.table[0, 3] = c.pools[0].shape[0]
    c.table[0, 0] = 2 ** 32 - 1
    c.table[1, :] = c.pools[0].shape[0] + 7
    c.table[3] = c.table[2]
    c.upload()
    q = rng.standard_normal((4, 4 * 64)).astype(np.float32)
    got = check(gpu, c, q, 4, weigh=True)
    assert (got[1] == 0).all()
    check(gpu, c, q, 4, length=[2 ** 32 - 1, 9, 161, 2 ** 31], weigh=True)
    check(gpu, c, q, 4, length=[10, 0, 1, 0], weigh=True)


@pytest.mark.parametrize("kind", KINDS)
def test_scores_far_apart(gpu, kind):
    """Scores of thousands, one row taking everything, rows of equal scores, and queries of very
    small and large values."""
    rng = np.random.default_rng(8)
    c = Paged(gpu, rng, kind, 2, 64, 16, [200, 33], gain=4.0)
    for scale in (1e-30, 1e-6, 30.0, 1e3):
        q = (scale * rng.standard_normal((2, 4 * 64))).astype(np.float32)
        check(gpu, c, q, 4, weigh=True)
    q[:] = 0.0
    check(gpu, c, q, 4, weigh=True)
    q = rng.standard_normal((2, 4 * 64)).astype(np.float32)
    q[:, ::7] *= 1e-5
    q[:, 3] = 3000.0
    check(gpu, c, q, 4, weigh=True)


@pytest.mark.parametrize("side", ["k", "v", "q"])
@pytest.mark.parametrize("kind", KINDS)
def test_a_nan_reaches_only_those_who_see_it(gpu, kind, side):
    rng = np.random.default_rng(9)
    n_head, n_kv, hd = 8, 2, 64
    c = Paged(gpu, rng, kind, n_kv, hd, 16, [150, 150, 40])
    q = rng.standard_normal((3, n_head * hd)).astype(np.float32)
    clean = check(gpu, c, q, n_head)
    bad = np.zeros((3, n_head, hd), bool)
    if side == "q":
        q[1, 3 * hd + 5] = np.nan
        bad[1, 3] = True
    else:
        c.pools[side == "v"][c.table[1, 100 // 16], 1, 100 % 16, 7] = NAN[kind]
        bad[1, 4:] = True
        if side == "v":
            bad[1, 4:, :7], bad[1, 4:, 8:] = False, False
        c.upload()
    got = attend(gpu, c, q, n_head)
    bad = bad.reshape(3, -1)
    assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], clean[~bad])
    assert np.array_equal(attend(gpu, c, q, n_head, length=[150, 100, 40])[[0, 2]], got[[0, 2]], equal_nan=True)


def test_the_same_every_time(gpu):
    """Sums in a fixed order: two calls give equal bits, weights too."""
    rng = np.random.default_rng(10)
    c = Paged(gpu, rng, rf.F16, 4, 128, 32, [3000, 17, 900])
    q = rng.standard_normal((3, 16 * 128)).astype(np.float32)
    a = attend(gpu, c, q, 16, weigh=True)
    wa = c.d_weight.numpy()
    c.upload()
    assert np.array_equal(a, attend(gpu, c, q, 16, weigh=True)) and np.array_equal(wa, c.d_weight.numpy())


# ---------------------------------------------------------------- eviction

EVICTS = [  # kv heads, head_dim, page, lengths, keep, recent
    (8, 128, 16, [129, 128, 127, 300], 128, 16), (2, 48, 16, [50, 1, 0, 49], 49, 0), (1, 256, 32, [2500], 1, 1),
    (3, 40, 64, [1000, 999], 998, 998), (2, 64, 16, [700, 10, 1500], 333, 100), (1, 8, 16, [5000], 2500, 0),
    (2, 96, 128, [4097], 1024, 7), (2, 64, 16, [40, 80], 1000, 5), (1, 16, 16, [20000], 300, 33)]


@pytest.mark.parametrize("values", ["spread", "equal", "odd"])
@pytest.mark.parametrize("case", EVICTS, ids=str)
@pytest.mark.parametrize("kind", KINDS)
def test_evict(gpu, kind, case, values):
    n_kv, hd, page, lengths, keep, recent = case
    rng = np.random.default_rng(len(values) + hd)
    c = Paged(gpu, rng, kind, n_kv, hd, page, lengths, room=20)
    c.weight[:] = np.exp(3 * rng.standard_normal(c.weight.shape))
    if values == "equal":
        c.weight[:] = rng.integers(0, 3, c.weight.shape)
    if values == "odd":
        c.weight[rng.random(c.weight.shape) < 0.2] = 0.0
        for x in (np.nan, np.inf, -1.0, 1e-44, -np.inf, -0.0):
            c.weight[rng.random(c.weight.shape) < 0.05] = x
    for s, n in enumerate(lengths):
        for h in range(n_kv):
            c.position[s, h, :n] = rng.permutation(n) + 5 * s
            c.position[s, h, n:] = 2 ** 32 - 1
    c.upload()
    kept = dev(gpu, np.full(len(lengths), 77, np.uint32))
    gpu.paged_evict(c.c, c.d_length, kept, keep, recent)
    k, v, w, p, m = pr.evict(*c.pools, c.table, c.weight, c.position, c.length, keep, recent)
    assert np.array_equal(kept.numpy(), m)
    assert np.array_equal(c.d_position.numpy(), p)
    assert np.array_equal(c.d_weight.numpy(), w, equal_nan=True)
    assert np.array_equal(c.k.numpy(), k) and np.array_equal(c.v.numpy(), v)
    # once more, of what is left: nothing moves
    c.length = m
    gpu.paged_evict(c.c, dev(gpu, m), kept, keep, recent)
    assert np.array_equal(c.k.numpy(), k) and np.array_equal(kept.numpy(), m)


@pytest.mark.parametrize("cap", [400, 5000, 40000])
@pytest.mark.parametrize("equal", [False, True])
def test_evict_by_ones_and_twos(gpu, cap, equal):
    """From one row too many to a dozen, in caches with little and much room, in keys all equal too."""
    rng = np.random.default_rng(cap)
    for keep in (1, 2, 5, 63, 64, 65, 380):
        lengths = [keep + x for x in range(0, 13)]
        c = Paged(gpu, rng, rf.F16, 1, 16, 16, lengths, room=cap - max(lengths))
        if equal:
            c.weight[:] = rng.integers(0, 2, c.weight.shape)
        for s, n in enumerate(lengths):
            c.position[s, 0, :n] = rng.permutation(n)
        c.upload()
        kept = dev(gpu, np.zeros(len(lengths), np.uint32))
        gpu.paged_evict(c.c, c.d_length, kept, keep, min(keep, 3))
        k, v, w, p, m = pr.evict(*c.pools, c.table, c.weight, c.position, c.length, keep, min(keep, 3))
        assert np.array_equal(kept.numpy(), m)
        assert np.array_equal(c.d_position.numpy(), p) and np.array_equal(c.d_weight.numpy(), w)
        assert np.array_equal(c.k.numpy(), k) and np.array_equal(c.v.numpy(), v)


@pytest.mark.parametrize("values", ["spread", "equal"])
@pytest.mark.parametrize("keep,recent", [(59999, 100), (59000, 0), (30000, 30000), (24576, 77), (100, 5), (1, 0)])
def test_evict_longer_than_registers(gpu, keep, recent, values):
    """Rows past those that a workgroup holds, read anew in every turn."""
    rng = np.random.default_rng(keep)
    c = Paged(gpu, rng, rf.BF16, 1, 8, 128, [60000, 24577, 24576], spare=0)
    c.weight[:] = np.exp(2 * rng.standard_normal(c.weight.shape)) if values == "spread" else \
        rng.integers(0, 2, c.weight.shape)
    for s, n in enumerate(c.length):
        c.position[s, 0, :n] = rng.permutation(int(n))
    c.upload()
    kept = dev(gpu, np.zeros(3, np.uint32))
    gpu.paged_evict(c.c, c.d_length, kept, keep, recent)
    k, v, w, p, m = pr.evict(*c.pools, c.table, c.weight, c.position, c.length, keep, recent)
    assert np.array_equal(kept.numpy(), m)
    assert np.array_equal(c.d_position.numpy(), p) and np.array_equal(c.d_weight.numpy(), w)
    assert np.array_equal(c.k.numpy(), k) and np.array_equal(c.v.numpy(), v)


@pytest.mark.parametrize("cap", [320, 5008, 9008])
@pytest.mark.parametrize("keep", [127, 128, 129])
def test_evict_mostly_the_newest(gpu, keep, cap):
    """Nearly all of the rows kept are the newest, and as many move as one launch takes, one less and one more."""
    rng = np.random.default_rng(keep + cap)
    for recent in (keep, keep - 1, keep - 30):
        c = Paged(gpu, rng, rf.F16, 2, 40, 16, [2 * keep + 20, keep + 9, 2 * keep], room=cap - 2 * keep - 20)
        for s, n in enumerate(c.length):
            c.position[s, :, :n] = np.arange(n)
        c.upload()
        kept = dev(gpu, np.zeros(3, np.uint32))
        gpu.paged_evict(c.c, c.d_length, kept, keep, recent)
        k, v, w, p, m = pr.evict(*c.pools, c.table, c.weight, c.position, c.length, keep, recent)
        assert np.array_equal(kept.numpy(), m)
        assert np.array_equal(c.d_position.numpy(), p) and np.array_equal(c.d_weight.numpy(), w)
        assert np.array_equal(c.k.numpy(), k) and np.array_equal(c.v.numpy(), v)


def test_evict_positions_alike_or_far(gpu):
    """Positions that say nothing (all the same, more of the newest than are kept, past 2^31): still
    `keep` rows, and nothing out of place."""
    rng = np.random.default_rng(11)
    c = Paged(gpu, rng, rf.F16, 2, 64, 16, [90, 90, 90])
    c.position[0] = 4
    c.position[1] = 2 ** 32 - 1 - rng.integers(0, 3, c.position[1].shape)
    c.position[2] = rng.integers(0, 2 ** 32, c.position[2].shape)
    c.upload()
    kept = dev(gpu, np.zeros(3, np.uint32))
    gpu.paged_evict(c.c, c.d_length, kept, 40, 30)
    k, v, w, p, m = pr.evict(*c.pools, c.table, c.weight, c.position, c.length, 40, 30)
    assert np.array_equal(c.k.numpy(), k) and np.array_equal(c.v.numpy(), v)
    assert np.array_equal(c.d_weight.numpy(), w) and np.array_equal(c.d_position.numpy(), p)


def test_evict_without_pages(gpu):
    """Rows that have no page move in the arrays only."""
    rng = np.random.default_rng(12)
    c = Paged(gpu, rng, rf.BF16, 1, 64, 16, [160])
    c.table[0, 1], c.table[0, 7] = c.pools[0].shape[0], 2 ** 32 - 1
    c.position[0, 0] = rng.permutation(c.cap)
    c.upload()
    kept = dev(gpu, np.zeros(1, np.uint32))
    gpu.paged_evict(c.c, c.d_length, kept, 60, 8)
    k, v, w, p, m = pr.evict(*c.pools, c.table, c.weight, c.position, c.length, 60, 8)
    assert np.array_equal(c.k.numpy(), k) and np.array_equal(c.v.numpy(), v)
    assert np.array_equal(c.d_weight.numpy(), w) and np.array_equal(c.d_position.numpy(), p)


# ------------------------------------------------------------ as they are used

class Server:
    """Three sequences decoded together with a budget of rows, step by step on the GPU; the numpy
    side takes the GPU's rows (their rounding is tested above) and its weights' order."""

    def __init__(self, gpu, kind, seed):
        self.rng = rng = np.random.default_rng(seed)
        self.gpu, self.n_head, self.n_kv, self.hd, self.budget = gpu, 8, 2, 64, 40
        self.c = Paged(gpu, rng, kind, 2, 64, 16, [37, 12, 40], room=8)
        for s, n in enumerate(self.c.length):
            self.c.position[s, :, :n] = np.arange(n)
        self.c.upload()
        n = 200
        cos, sin = gpu.empty((n, 32), np.float32), gpu.empty((n, 32), np.float32)
        gpu.rope_tables(cos, sin, n, 64, base=10000.0, scale=0.5)
        self.cos, self.sin, self.n_table = cos, sin, n
        self.pos = np.array([37, 12, 50], np.uint32)     # (the third was cut back before)
        e = lambda *s: gpu.empty(s, np.float32)
        self.q, self.qo, self.out, self.k, self.v = e(3, 512), e(3, 512), e(3, 512), e(3, 128), e(3, 128)
        self.d_pos, self.d_row, self.d_len = (gpu.empty(3, np.uint32) for _ in range(3))
        self.kept = gpu.empty(3, np.uint32)

    def inputs(self):
        q, k, v = (self.rng.standard_normal(s).astype(np.float32) for s in ((3, 512), (3, 128), (3, 128)))
        self.hq = q
        self.q.upload(q)
        self.k.upload(k)
        self.v.upload(v)
        self.d_pos.upload(self.pos)
        self.d_row.upload(self.c.length)
        self.d_len.upload(self.c.length + 1)

    def calls(self):
        g, c = self.gpu, self.c.c
        g.paged_rope_store(c, self.q, self.qo, 8, self.k, self.v, 3, self.d_pos, 64, rf.PAIRS_HALVES, self.cos,
                           self.sin, self.n_table, row=self.d_row)
        g.paged_attention(c, self.out, self.qo, 8, 3, self.d_len, weigh=True)
        g.paged_evict(c, self.d_len, self.kept, self.budget, 8)

    def step(self, launch):
        c = self.c
        before = [c.k.numpy(), c.v.numpy()]
        self.inputs()
        launch()
        length = c.length + 1
        # the rows just stored: rows of the pools before the eviction moved any
        at = c.table[np.arange(3), c.length // 16], c.length % 16
        cos, sin = self.cos.numpy()[self.pos], self.sin.numpy()[self.pos]
        want, _ = pr.norm_rope(self.hq, 64, None, 0, cos, sin, 1, 64)
        q = self.qo.numpy()
        assert np.abs(q - want).max() < 1e-5
        wk, _ = pr.norm_rope(self.k.numpy(), 64, None, 0, cos, sin, 1, 64)
        for pool, x in zip(before, (wk, self.v.numpy())):
            pool[at[0], :, at[1]] = pr.to_bits(x, c.kind).reshape(3, 2, 64)
        c.weight[np.arange(3), :, c.length], c.position[np.arange(3), :, c.length] = 0.0, self.pos[:, None]
        want, sizes, ps = pr.attention(q, *before, c.table, c.kind, 8, length, np.arange(3))
        assert (np.abs(self.out.numpy() - want) <= pr.attention_bound(sizes)).all()
        for s in range(3):
            for h in range(2):
                c.weight[s, h, :length[s]] += np.array(ps[s][4 * h:4 * h + 4]).sum(0).astype(np.float32)
        k, v, w, p, m = pr.evict(*before, c.table, c.weight, c.position, length, self.budget, 8)
        assert np.array_equal(self.kept.numpy(), m)
        assert np.array_equal(c.d_position.numpy(), p)
        assert np.array_equal(c.k.numpy(), k) and np.array_equal(c.v.numpy(), v)
        assert np.abs(c.d_weight.numpy() - w).max() < 1e-4
        c.weight, c.position, c.length = c.d_weight.numpy(), p, m
        self.pos = self.pos + 1


@pytest.mark.parametrize("kind", KINDS)
def test_steps_of_a_server(gpu, kind):
    s = Server(gpu, kind, 20)
    for _ in range(12):
        s.step(s.calls)


def test_captured_steps(gpu):
    """The step as one graph, replayed with eager work between the replays."""
    import ctypes as C
    s = Server(gpu, rf.F16, 21)
    s.step(s.calls)
    g, lib = C.c_void_p(), gpu.lib
    assert lib.fox_gpu_graph_begin(gpu.ctx) == 0
    s.calls()
    assert lib.fox_gpu_graph_end(gpu.ctx, C.byref(g)) == 0

    def replay():
        assert lib.fox_gpu_graph_launch(gpu.ctx, g) == 0
    for i in range(6):
        s.step(replay)
        if i % 2:
            s.step(s.calls)
    gpu.sync()
    lib.fox_gpu_graph_free(g)


def test_two_contexts_at_once(gpu):
    """Two contexts attend over one cache at the same time, and give what each gives alone."""
    rng = np.random.default_rng(22)
    c = Paged(gpu, rng, rf.BF16, 4, 128, 64, [2000, 700], track=False)
    q = rng.standard_normal((2, 16 * 128)).astype(np.float32)
    want = attend(gpu, c, q, 16)
    other = rf.Gpu(0)
    sides = [(g, dev(g, q), g.empty(q.shape, np.float32), dev(g, c.length)) for g in (gpu, other)]
    for _ in range(20):
        for g, dq, out, n in sides:
            g.paged_attention(c.c, out, dq, 16, 2, n)
    for g, dq, out, n in sides:
        assert np.array_equal(out.numpy(), want)
    for g, dq, out, n in sides[1:]:
        for a in (dq, out, n):
            a.free()
    other.close()


def test_pools_past_four_gigabytes(gpu):
    """Pages whose first element is past 2^32: stored, attended to, moved."""
    n_kv, hd, page, pages = 8, 128, 64, 70000
    per = n_kv * page * hd
    assert per * pages > 1 << 32
    rng = np.random.default_rng(23)
    pools = [gpu.empty(per * pages, np.uint16) for _ in range(2)]
    table = np.array([[69999, 0, 65536, 66000]], np.uint32)
    weight = gpu.array(rng.random((1, n_kv, 256)).astype(np.float32))
    position = gpu.array(np.tile(np.arange(256, dtype=np.uint32), (1, n_kv, 1)))
    c = rf.PagedCache(rf.F16, *pools, pages, page, n_kv, hd, gpu.array(table), 1, 4, weight, position)
    M, w = 240, n_kv * hd
    k, v = (rng.standard_normal((M, w)).astype(np.float32) for _ in range(2))
    cos, sin = gpu.array(np.ones((M, 64), np.float32)), gpu.array(np.zeros((M, 64), np.float32))
    q = rng.standard_normal((M, w)).astype(np.float32)
    gpu.paged_rope_store(c, gpu.array(q), gpu.empty(q.shape, np.float32), n_kv, gpu.array(k), gpu.array(v), M,
                         gpu.array(np.arange(M, dtype=np.uint32)), hd, 0, cos, sin, M,
                         seq=gpu.array(np.zeros(M, np.uint32)))
    small = [np.zeros((4, n_kv, page, hd), np.uint16) for _ in range(2)]
    for x, p in zip((k, v), small):
        r = np.arange(M)
        p[r // page, :, r % page] = pr.to_bits(x, rf.F16).reshape(M, n_kv, hd)
    out = gpu.empty((1, w), np.float32)
    length = gpu.array(np.array([M], np.uint32))
    gpu.paged_attention(c, out, gpu.array(q[:1]), n_kv, 1, length)
    tab = np.arange(4, dtype=np.uint32)[None]
    want, sizes, _ = pr.attention(q[:1], *small, tab, rf.F16, n_kv, [M], [0])
    assert (np.abs(out.numpy() - want) <= pr.attention_bound(sizes)).all()
    hw, hp = weight.numpy(), position.numpy()
    kept = gpu.empty(1, np.uint32)
    gpu.paged_evict(c, length, kept, 100, 20)
    ek, ev, _, _, _ = pr.evict(*small, tab, hw, hp, [M], 100, 20)
    gpu.paged_attention(c, out, gpu.array(q[:1]), n_kv, 1, kept)
    want, sizes, _ = pr.attention(q[:1], ek, ev, tab, rf.F16, n_kv, [100], [0])
    assert (np.abs(out.numpy() - want) <= pr.attention_bound(sizes)).all()
    for p in pools:
        p.free()
