"""Timed cases of the paged caches: many sequences decoded together.

Four operators:

  table  cosines and sines of the positions' angles, as they are or scaled for contexts longer
         than the model was trained on (``Gpu.rope_tables``)
  rope   RMSNorm of every query and key head, the rotation of the first dimensions of each and
         the store of keys and values into the pages of the tokens' sequences
         (``Gpu.paged_rope_store``)
  attn   attention of one new token of every sequence over its pages, the softmax's weights
         added to those that the rows have got so far where asked for (``Gpu.paged_attention``)
  evict  of every sequence longer than a budget, each kv head keeps the newest rows and those
         that got the most weight (``Gpu.paged_evict``)

The cache.  Keys and values are two pools, [pages][kv heads][rows of a page][head_dim] in 16
bits; a table gives the pages of each sequence in order, taken from all over the pool as an
allocator leaves them.  Row r of a sequence is row r % page of its page r / page.  Beside the
pools stand two arrays [sequences][kv heads][rows]: the weight that a row got, and its token's
position.

Eviction.  Of a sequence's rows, every kv head keeps ``keep``: first those whose position is
above the head's greatest by less than -recent, then those of the greatest weight, of equal
ones the lower row.  Kept rows from ``keep`` on, in order, take the places of those that are not
kept below it, in order; the others stay where they are.

A decoder walks a stack of layers that do not fit the card's caches together; a state of the
attention holds several layers' pools, of the same contents, and successive passes take them in
turn.
"""
import math
from types import SimpleNamespace

import torch

own = False

EPS = 1e-6
BASE = 500000.0
TRAINED = 8192              # positions that the scaled tables' model was trained on
ROTATE = 600 << 20          # bytes of pools one state holds, about
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the smallest model's tables: a launch
        dict(name="table-tiny", op="table", scaling="none", rows=2048, n_rot=48),
        # tables of a 16 times longer context, slow pairs stretched and fast ones kept
        dict(name="table-long", op="table", scaling="ramp", rows=131072, n_rot=128),
        # a decode step of 32 sequences of the 8B class
        dict(name="rope-step-8b", op="rope", type="f16", pairs="adjacent", heads=32, kv_heads=8,
             head_dim=128, n_rot=128, norms=False, page=64, seqs=32, tokens=1, past=1500),
        # eight drafted tokens of five sequences, head norms, a part of the head turned
        dict(name="rope-part-5x8", op="rope", type="bf16", pairs="halves", heads=32, kv_heads=8,
             head_dim=128, n_rot=64, norms=True, page=16, seqs=5, tokens=8, past=333),
        # a prompt of the 27B class, an odd number of tokens
        dict(name="rope-prompt-27b", op="rope", type="bf16", pairs="halves", heads=32, kv_heads=16,
             head_dim=128, n_rot=128, norms=True, page=64, seqs=1, tokens=1001, past=0),
        # the smallest model's step, three sequences: bound by launches
        dict(name="attn-tiny-3", op="attn", type="f16", heads=6, kv_heads=6, head_dim=48, page=16,
             seqs=3, longest=35, ragged=True, weigh=False),
        # one answer token of the 8B class
        dict(name="attn-8b-1", op="attn", type="f16", heads=32, kv_heads=8, head_dim=128, page=64,
             seqs=1, longest=4097, ragged=False, weigh=False),
        # one answer token on a very long document
        dict(name="attn-4b-1-long", op="attn", type="bf16", heads=32, kv_heads=8, head_dim=128,
             page=128, seqs=1, longest=131071, ragged=False, weigh=False),
        # a server's step: sequences of unlike lengths, rows weighed
        dict(name="attn-8b-24-weigh", op="attn", type="f16", heads=32, kv_heads=8, head_dim=128,
             page=16, seqs=24, longest=6001, ragged=True, weigh=True),
        # the widest step
        dict(name="attn-27b-64", op="attn", type="bf16", heads=32, kv_heads=16, head_dim=128, page=32,
             seqs=64, longest=8192, ragged=True, weigh=False),
        # every step at its budget gives a row up for the new one
        dict(name="evict-step-8b", op="evict", type="f16", kv_heads=8, head_dim=128, page=16, seqs=16,
             longest=2049, keep=2048, recent=256, ragged=False),
        # conversations cut back to their budget, some of them below it
        dict(name="evict-turn-8b", op="evict", type="bf16", kv_heads=8, head_dim=128, page=64, seqs=6,
             longest=20011, keep=4096, recent=512, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(hi, lo))))))


def draw(rng):
    op = rng.choice(["table", "rope", "rope", "attn", "attn", "attn", "evict", "evict"])
    if op == "table":
        n_rot = 2 * rng.choice([12, 16, 20, 24, 32, 48, 64, 96, 128])
        return dict(op=op, scaling=rng.choice(["none", "linear", "ramp", "factors"]), n_rot=n_rot,
                    rows=_log_int(rng, 100, (131072 * 128) // n_rot))
    kv = rng.choice([1, 2, 4, 6, 8, 8, 16])
    hd = rng.choice([40, 48, 64, 80, 96, 128, 128, 128, 192, 256])
    kind, page = rng.choice(["f16", "bf16"]), rng.choice([16, 32, 64, 128])
    heads = kv * rng.choice([1, 2, 4] if kv > 8 else [1, 2, 4, 5, 8])
    if op == "rope":
        seqs = rng.choice([1, rng.randint(2, 8), rng.randint(9, 64)])
        tokens = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 1000)])
        tokens = max(1, min(tokens, 1000 // seqs))
        return dict(op=op, type=kind, pairs=rng.choice(["halves", "adjacent"]), heads=heads, kv_heads=kv,
                    head_dim=hd, n_rot=rng.choice([hd, hd, 8 * rng.randint(1, hd // 8)]),
                    norms=rng.random() < 0.5, page=page, seqs=seqs, tokens=tokens,
                    past=_log_int(rng, 1, max(1, (24 << 20) // (seqs * kv * hd))))
    if op == "attn":
        seqs = rng.choice([1, rng.randint(2, 8), _log_int(rng, 9, 96)])
        # (the largest listed case reads 4e8 values of each of its pools, for two heads each)
        most = (380 << 20) // max(1, heads // kv // 2)
        return dict(op=op, type=kind, heads=heads, kv_heads=kv, head_dim=hd, page=page, seqs=seqs,
                    longest=_log_int(rng, 1, min(131000, most // (seqs * kv * hd))),
                    ragged=rng.random() < 0.7, weigh=rng.random() < 0.35)
    seqs = rng.choice([1, rng.randint(2, 8), rng.randint(9, 32)])
    longest = _log_int(rng, 40, min(30000, (120 << 20) // (seqs * kv * hd)))
    keep = rng.choice([longest - 1, rng.randint(1, longest), max(1, longest // 4)])
    return dict(op=op, type=kind, kv_heads=kv, head_dim=hd, page=page, seqs=seqs, longest=longest,
                keep=keep, recent=rng.randint(0, keep), ragged=rng.random() < 0.5)


def _lengths(case):
    """Rows of each sequence: all as long as the longest, or from a twentieth of it up."""
    n, most = case["seqs"], case["longest"]
    if not case["ragged"]:
        return [most] * n
    u = [(0.618034 * i) % 1.0 for i in range(n)]
    return [most if i == 0 else max(1, int(most * (0.05 + 0.95 * u[i] * u[i]))) for i in range(n)]


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


class _Dev:
    """A torch tensor under the name the package's calls use."""

    def __init__(self, t):
        self.t = t.contiguous()
        self.ptr = self.t.data_ptr()


_context = None


def _gpu():
    global _context
    if _context is None:
        import rustfox_amd as rf
        _context = rf.Gpu(0)
    return _context


def _u32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pools(g, case, pages):
    """Keys with channels of unequal size, so that the weights are uneven, and values."""
    kvh, hd, page, kind = case["kv_heads"], case["head_dim"], case["page"], TYPES[case["type"]]
    gain = torch.exp(0.5 * _randn(g, kvh, 1, hd))
    k = torch.empty(pages, kvh, page, hd, dtype=kind, device="cuda")
    v = torch.empty_like(k)
    step = max(1, (1 << 26) // (kvh * page * hd))
    for i in range(0, pages, step):
        n = min(step, pages - i)
        k[i:i + n] = _randn(g, n, kvh, page, hd) * gain
        v[i:i + n] = 0.5 * _randn(g, n, kvh, page, hd)
    return k, v


def _table(g, seqs, most, page):
    """[seqs][pages of a sequence] places in the pool, in no order."""
    per = -(-most // page)
    at = torch.randperm(seqs * per, generator=g, device="cuda")
    return at.reshape(seqs, per).to(torch.int32)


def _scaling(case):
    """What rope_tables takes, and the pairs' divisors."""
    n = case["n_rot"] // 2
    if case["scaling"] == "linear":
        return dict(base=BASE, scale=0.25), None
    if case["scaling"] == "ramp":
        return dict(base=BASE, scale=1.0 / 16, ext=1.0, beta_fast=32.0, beta_slow=1.0, orig_ctx=TRAINED,
                    magnitude=1.0 + 0.1 * math.log(16.0)), None
    if case["scaling"] == "factors":
        return dict(base=BASE), torch.linspace(0.0, 3.0, n, dtype=torch.float64).exp().float().cuda()
    return dict(base=BASE), None


def _plain_tables(n, n_rot, base=BASE):
    ex = base ** (-2.0 * torch.arange(n_rot // 2, dtype=torch.float64) / n_rot)
    th = torch.arange(n, dtype=torch.float64)[:, None] * ex
    return th.cos().float().cuda(), th.sin().float().cuda()


def _inputs(case, seed):
    """Everything random that a case starts from; the same values each time."""
    g, s = _gen(seed), SimpleNamespace()
    kvh, hd, page, seqs = (case[x] for x in ("kv_heads", "head_dim", "page", "seqs"))
    if case["op"] == "rope":
        M, heads = seqs * case["tokens"], case["heads"]
        first = [max(0, case["past"] - 7 * i) for i in range(seqs)]
        s.most = case["past"] + case["tokens"]
        s.pos = [p + t for p in first for t in range(case["tokens"])]
        s.seq = [i for i in range(seqs) for _ in range(case["tokens"])]
        s.q = 1.5 * _randn(g, M, heads * hd)
        s.new_k, s.new_v = _randn(g, M, kvh * hd), 0.5 * _randn(g, M, kvh * hd)
        s.qn, s.kn = (1.0 + 0.1 * _randn(g, hd) for _ in range(2)) if case["norms"] else (None, None)
        s.cos, s.sin = _plain_tables(s.most, case["n_rot"])
    else:
        s.length = _lengths(case)
        s.most = case["longest"]
    s.table = _table(g, seqs, s.most, page)
    s.cap = s.table.shape[1] * page
    s.k, s.v = _pools(g, case, s.table.numel())
    if case["op"] == "attn":
        s.q = 1.5 * _randn(g, seqs, case["heads"] * hd)
        if case["weigh"]:
            s.weight = torch.rand(seqs, kvh, s.cap, generator=g, device="cuda")
    if case["op"] == "evict":
        # (new rows have no weight yet; what earlier evictions moved is in no order)
        s.weight = torch.exp(2.0 * _randn(g, seqs, kvh, s.cap))
        s.weight[torch.rand(seqs, kvh, s.cap, generator=g, device="cuda") < 0.03] = 0.0
        s.position = torch.zeros(seqs, kvh, s.cap, dtype=torch.int32, device="cuda")
        for i, n in enumerate(s.length):
            s.position[i, :, :n] = torch.rand(kvh, n, generator=g, device="cuda").argsort(-1).to(torch.int32)
    return s


def prepare(case, seed):
    if case["op"] == "table":
        s = SimpleNamespace(case=case, own=own, turn=0)
        # (another seed's tables begin at another position)
        s.p0 = seed % 97
        s.how, s.factors = _scaling(case)
        s.cos, s.sin = (_Dev(torch.zeros(case["rows"], case["n_rot"] // 2, device="cuda")) for _ in range(2))
        if own:
            s.gpu = _gpu()
            s.f = _Dev(s.factors) if s.factors is not None else None
        torch.cuda.synchronize()
        return s
    s = _inputs(case, seed)
    s.case, s.own, s.turn = case, own, 0
    size = 2 * s.k.numel() * s.k.element_size()
    n = max(1, min(16, ROTATE // size)) if case["op"] == "attn" else 1
    s.pools = [(s.k, s.v)] + [(s.k.clone(), s.v.clone()) for _ in range(n - 1)]
    if case["op"] != "evict":
        s.out = torch.zeros_like(s.q)
    track = case["op"] == "evict" or case.get("weigh", False)
    if track:
        # weights, then positions, in one piece; and as they are before a pass
        at = s.weight.numel()
        s.before = torch.zeros(2 * at, device="cuda")
        s.before[:at] = s.weight.reshape(-1)
        if case["op"] == "evict":
            s.before[at:] = s.position.reshape(-1).view(torch.float32)
        s.track = s.before.clone()
        s.weight = s.track[:at].view(s.weight.shape)
        s.position = s.track[at:].view(torch.int32).view(s.weight.shape)
    if case["op"] == "rope":
        s.pos, s.seq = _u32(s.pos), _u32(s.seq)
    else:
        s.length = _u32(s.length)
    if case["op"] == "evict":
        s.kept = torch.zeros_like(s.length)
    if own:
        import rustfox_amd as rf
        s.gpu = _gpu()
        kind = rf.F16 if case["type"] == "f16" else rf.BF16
        s.d = SimpleNamespace(**{x: _Dev(t) for x, t in vars(s).items() if isinstance(t, torch.Tensor)})
        s.caches = [rf.PagedCache(kind, _Dev(k), _Dev(v), s.table.numel(), case["page"], case["kv_heads"],
                                  case["head_dim"], s.d.table, case["seqs"], s.table.shape[1],
                                  s.d.weight if track else None, s.d.position if track else None)
                    for k, v in s.pools]
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------ the operators

def run(s):
    s.turn += 1
    return (_run_own if s.own else _run_plain)(s)


def _outputs(s, k, v):
    op = s.case["op"]
    if op == "table":
        return [s.cos.t, s.sin.t]
    if op == "rope":
        return [s.out, k, v]
    if op == "attn":
        return [s.out, s.weight] if s.case["weigh"] else s.out
    return [k, v, s.weight, s.position, s.kept]


def _run_own(s):
    c = s.case
    if c["op"] == "table":
        s.gpu.rope_tables(s.cos, s.sin, c["rows"], c["n_rot"], p0=s.p0, factors=s.f, **s.how)
        return _outputs(s, None, None)
    i = s.turn % len(s.pools)
    cache, d = s.caches[i], s.d
    if c["op"] == "rope":
        import rustfox_amd as rf
        pairs = rf.PAIRS_HALVES if c["pairs"] == "halves" else rf.PAIRS_ADJACENT
        norms = dict(q_norm=d.qn, k_norm=d.kn, eps=EPS) if c["norms"] else {}
        s.gpu.paged_rope_store(cache, d.q, d.out, c["heads"], d.new_k, d.new_v, c["seqs"] * c["tokens"],
                               d.pos, c["n_rot"], pairs, d.cos, d.sin, s.most,
                               seq=None if c["tokens"] == 1 else d.seq, **norms)
    else:
        if c["op"] == "evict" or c["weigh"]:
            s.gpu.copy(d.track, d.before, 4 * s.before.numel())
        if c["op"] == "attn":
            s.gpu.paged_attention(cache, d.out, d.q, c["heads"], c["seqs"], d.length, weigh=c["weigh"])
        else:
            s.gpu.paged_evict(cache, d.length, d.kept, c["keep"], c["recent"])
    return _outputs(s, *s.pools[i])


def _frequencies(case):
    """[n_rot / 2] angles of a position, in 64 bits, and the factor of every cosine and sine."""
    how, factors = _scaling(case)
    n = case["n_rot"]
    j = torch.arange(n // 2, dtype=torch.float64, device="cuda")
    f = how["base"] ** (-2.0 * j / n)
    if factors is not None:
        f = f / factors.double()
    mix = torch.zeros_like(f) if "scale" in how else torch.ones_like(f)
    if "ext" in how:
        at = [n * math.log(how["orig_ctx"] / (2 * math.pi * b)) / (2 * math.log(how["base"]))
              for b in (how["beta_fast"], how["beta_slow"])]
        lo, hi = max(0, math.floor(at[0])), min(n - 1, math.ceil(at[1]))
        mix = how["ext"] * (1.0 - ((j - lo) / max(0.001, hi - lo)).clamp(0.0, 1.0))
    return f * (how.get("scale", 1.0) * (1.0 - mix) + mix), how.get("magnitude", 1.0)


def _norm_rope(x, heads, hd, w, cos, sin, pairs, n_rot):
    """In 64 bits: a 16-bit key next to a border depends on the last bits."""
    x = x.double().reshape(-1, heads, hd)
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
    c, s = cos.double()[:, None, :], sin.double()[:, None, :]
    r, rest = x[..., :n_rot], x[..., n_rot:]
    a, b = (r[..., :n_rot // 2], r[..., n_rot // 2:]) if pairs == "halves" else (r[..., ::2], r[..., 1::2])
    ra, rb = a * c - b * s, a * s + b * c
    y = torch.cat([ra, rb], -1) if pairs == "halves" else torch.stack([ra, rb], -1).flatten(-2)
    return torch.cat([y, rest], -1).flatten(1).float()


def _held(x, kind):
    """16-bit values of floats; halves end at 65504."""
    return (x.clamp(-65504.0, 65504.0) if kind == torch.float16 else x).to(kind)


def _run_plain(s):
    c = s.case
    if c["op"] == "table":
        w, mag = _frequencies(c)
        p = torch.arange(s.p0, s.p0 + c["rows"], dtype=torch.float64, device="cuda")
        th = p[:, None] * w
        s.cos.t.copy_(mag * th.cos())
        s.sin.t.copy_(mag * th.sin())
        return _outputs(s, None, None)
    k, v = s.pools[s.turn % len(s.pools)]
    kvh, hd, page, seqs = (c[x] for x in ("kv_heads", "head_dim", "page", "seqs"))
    if c["op"] == "rope":
        at = s.pos.long()
        cos, sin = s.cos[at], s.sin[at]
        s.out.copy_(_norm_rope(s.q, c["heads"], hd, s.qn, cos, sin, c["pairs"], c["n_rot"]))
        key = _norm_rope(s.new_k, kvh, hd, s.kn, cos, sin, c["pairs"], c["n_rot"])
        pg = s.table[s.seq.long(), at // page].long()
        k[pg, :, at % page] = _held(key, k.dtype).reshape(-1, kvh, hd)
        v[pg, :, at % page] = _held(s.new_v, v.dtype).reshape(-1, kvh, hd)
        return _outputs(s, k, v)
    if c["op"] == "evict" or c["weigh"]:
        s.track.copy_(s.before)
    rows = torch.arange(s.cap, device="cuda")
    if c["op"] == "attn":
        heads, n = c["heads"], s.cap
        kk = k[s.table.long()].permute(0, 2, 1, 3, 4).reshape(seqs * kvh, n, hd).float()
        vv = v[s.table.long()].permute(0, 2, 1, 3, 4).reshape(seqs * kvh, n, hd).float()
        q = s.q.reshape(seqs * kvh, heads // kvh, hd)
        sc = torch.matmul(kk, q.transpose(1, 2).contiguous()).transpose(1, 2) * (1.0 / math.sqrt(hd))
        hidden = (rows[None] >= s.length[:, None]).repeat_interleave(kvh, 0)
        sc = sc.masked_fill(hidden[:, None, :], -math.inf)
        e = torch.exp(sc - sc.amax(-1, keepdim=True))
        p = e / e.sum(-1, keepdim=True)
        s.out.copy_(torch.matmul(p, vv).reshape(seqs, heads * hd))
        if c["weigh"]:
            s.weight += p.sum(1).reshape(seqs, kvh, n)
        return _outputs(s, k, v)
    keep, n = c["keep"], s.length[:, None, None]
    live = rows < n
    newest = s.position.masked_fill(~live, -1).amax(-1, keepdim=True)
    key = torch.where(s.position > newest - c["recent"], math.inf, s.weight).masked_fill(~live, -1.0)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.zeros_like(live.expand(key.shape)).scatter_(-1, order, True)
    kept = torch.where(n > keep, kept, live)
    si, hi, to = torch.nonzero(~kept & (rows < keep) & (n > keep), as_tuple=True)
    _, _, fr = torch.nonzero(kept & (rows >= keep) & (n > keep), as_tuple=True)
    pt, pf = (s.table[si, x // page].long() for x in (to, fr))
    for t in (k, v):
        t[pt, hi, to % page] = t[pf, hi, fr % page]
    for t in (s.weight, s.position):
        t[si, hi, to] = t[si, hi, fr]
    s.kept.copy_(s.length.clamp(max=keep))
    return _outputs(s, k, v)


# ------------------------------------------------------------ what it takes

def work(case):
    op = case["op"]
    if op == "table":
        n = case["rows"] * case["n_rot"] // 2
        return {"bytes": 8 * n, "flops": 30 * n}
    kvh, hd = case["kv_heads"], case["head_dim"]
    if op == "rope":
        M, nq, nkv = case["seqs"] * case["tokens"], case["heads"] * hd, kvh * hd
        return {"bytes": M * (8 * nq + 8 * nkv + 4 * nkv + 4 * case["n_rot"]), "flops": 10 * M * (nq + nkv)}
    rows = sum(_lengths(case))
    if op == "attn":
        weights = 8 * rows * kvh if case["weigh"] else 0
        return {"bytes": 4 * rows * kvh * hd + weights + 8 * case["seqs"] * case["heads"] * hd,
                "flops": 4 * rows * case["heads"] * hd}
    cut = [n for n in _lengths(case) if n > case["keep"]]
    # (weights know nothing of rows: the kept ones lie evenly)
    moved = sum(case["keep"] * (n - case["keep"]) // n for n in cut) * kvh
    return {"bytes": 8 * sum(cut) * kvh + moved * (8 * hd + 16), "flops": 2 * sum(cut) * kvh}


# ------------------------------------------------------------- in 64 bits

def _angles(case, p):
    """Angles of positions p [n], in 64 bits, and the magnitude: pair by pair."""
    how, factors = _scaling(case)
    n = case["n_rot"]
    out = torch.empty(p.numel(), n // 2, dtype=torch.float64, device="cuda")
    for j in range(n // 2):
        w = math.exp(-2.0 * j / n * math.log(how["base"]))
        if factors is not None:
            w /= float(factors[j])
        if case["scaling"] == "linear":
            w *= how["scale"]
        if case["scaling"] == "ramp":
            turn = [how["orig_ctx"] / (2 * math.pi * how["beta_" + x]) for x in ("fast", "slow")]
            lo, hi = (n / 2 * math.log(t) / math.log(how["base"]) for t in turn)
            lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), n - 1)
            part = min(1.0, max(0.0, (j - lo) / max(hi - lo, 0.001)))
            w = part * how["scale"] * w + (1.0 - part) * w
        out[:, j] = p * w
    return out, how.get("magnitude", 1.0)


def exact(case, seed):
    op = case["op"]
    if op == "table":
        th, mag = _angles(case, torch.arange(case["rows"], dtype=torch.float64, device="cuda") + seed % 97)
        return [mag * torch.cos(th), mag * torch.sin(th)]
    s = _inputs(case, seed)
    kvh, hd, page, seqs = (case[x] for x in ("kv_heads", "head_dim", "page", "seqs"))
    if op == "rope":
        heads, n_rot = case["heads"], case["n_rot"]
        q, key = s.q.double(), s.new_k.double()
        at = torch.tensor(s.pos, device="cuda")
        cos, sin = s.cos[at].double(), s.sin[at].double()
        for x, nh, w in ((q, heads, s.qn), (key, kvh, s.kn)):
            for h in range(nh):
                one = x[:, h * hd:(h + 1) * hd]
                if w is not None:
                    one *= w.double() * (one.pow(2).sum(-1, keepdim=True) / hd + EPS).rsqrt()
                for j in range(n_rot // 2):
                    i, m = (j, j + n_rot // 2) if case["pairs"] == "halves" else (2 * j, 2 * j + 1)
                    a, b = one[:, i].clone(), one[:, m].clone()
                    one[:, i] = a * cos[:, j] - b * sin[:, j]
                    one[:, m] = b * cos[:, j] + a * sin[:, j]
        for t, x in ((s.k, key.float()), (s.v, s.new_v)):
            # (a key is rounded to a float before it is rounded to 16 bits)
            rows = _held(x, t.dtype).reshape(-1, kvh, hd)
            for i, (sq, p) in enumerate(zip(s.seq, s.pos)):
                t[int(s.table[sq, p // page]), :, p % page] = rows[i]
        return [q, s.k, s.v]
    if op == "attn":
        heads, g = case["heads"], case["heads"] // kvh
        if sum(s.length) * heads * hd > 6e10:
            return None
        out = torch.empty(seqs, heads * hd, dtype=torch.float64, device="cuda")
        weight = s.weight.double() if case["weigh"] else None
        for i, n in enumerate(s.length):
            pg = s.table[i, :-(-n // page)].long()
            for h in range(kvh):
                kk = s.k[pg, h].reshape(-1, hd)[:n].double()
                vv = s.v[pg, h].reshape(-1, hd)[:n].double()
                for u in range(h * g, (h + 1) * g):
                    p = torch.softmax(torch.mv(kk, s.q[i, u * hd:(u + 1) * hd].double()) / math.sqrt(hd), 0)
                    out[i, u * hd:(u + 1) * hd] = torch.mv(vv.t().contiguous(), p)
                    if weight is not None:
                        weight[i, h, :n] += p
        return [out, weight] if case["weigh"] else out
    keep = case["keep"]
    for i, n in enumerate(s.length):
        if n <= keep:
            continue
        row = torch.arange(n, device="cuda")
        where = s.table[i].long()[row // page] * kvh * page + row % page      # of kv head 0
        for h in range(kvh):
            pos, w = s.position[i, h, :n], s.weight[i, h, :n]
            new = pos > pos.max() - case["recent"]
            # by weight, rows of equal weight in order: the newest stand before all
            order = torch.argsort(torch.where(new, torch.full_like(w, math.inf), w), descending=True, stable=True)
            chosen, _ = torch.sort(order[:keep])
            inside = torch.zeros(n, dtype=torch.bool, device="cuda")
            inside[chosen] = True
            hole, late = row[:keep][~inside[:keep]], chosen[chosen >= keep]
            for t in (s.k, s.v):
                flat = t.view(-1, hd)
                flat[where[hole] + h * page] = flat[where[late] + h * page]
            pos[hole], w[hole] = pos[late], w[late]
    return [s.k, s.v, s.weight, s.position, torch.tensor([min(n, keep) for n in s.length], dtype=torch.int32)]
