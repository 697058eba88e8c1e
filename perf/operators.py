"""Timed cases of the quantised caches and the attention that reads them.

Three operators on one sequence's cache:

  kv     rows quantised into a cache as they are written (``Gpu.kvq_write``) and rows read
         back as floats (``Gpu.kvq_read``)
  rope   RMSNorm of every query and key head, the position rotation and the store of keys
         and values, in the float caches (``Gpu.norm_rope_store``) or a quantised one
         (``Gpu.kvq_norm_rope_store``)
  attn   causal attention of the tokens at positions past .. past + tokens - 1 over a
         quantised cache (``Gpu.kvq_attention``)

The format.  A head's dimensions are quantised in groups of 32 (the last group of a head may
be shorter), 4 or 8 bits a value, with one 8-bit scale for a group: an unsigned number of
5 exponent and 3 mantissa bits, (8 + m) 2^e or m 2^-19 at the lowest exponent.  A group's scale is the
smallest one with max <= (h - 1/2) d and -min <= (h + 1/2) d, h = 8 or 128, at most 224
(4 bits) or 120 (8 bits); a value's code is x / d rounded to the nearest integer, ties to
even, within [-h, h - 1].

Keys have channels of unequal size and queries are N(0, 1.5), so that the weights of the
softmax are uneven, as a model's are.  A decoder walks a stack of layers that do not fit the
card's caches together; a state holds several layers' caches, of the same contents, and
successive passes take them in turn.
"""
import math
from types import SimpleNamespace

import torch

own = False

EPS = 1e-6
BASE = 10000.0
HALF = {4: 8, 8: 128}       # codes are within [-HALF, HALF - 1]
CAP = {4: 224.0, 8: 120.0}  # largest scale
ROTATE = 90 << 20           # bytes of caches one state holds, about


def listed():
    return [
        # a decode step's new row of the 8B class, stored and fetched: two small launches
        dict(name="kv-step-8b", op="kv", bits=4, kv_heads=8, head_dim=128, past=4095, tokens=1,
             first=4095),
        # a prompt's rows of the 27B class, an odd number of them, from an odd position
        dict(name="kv-prompt-27b", op="kv", bits=4, kv_heads=16, head_dim=128, past=333,
             tokens=1001, first=333),
        # a session handed on: its last rows stored, the whole cache read back as floats
        dict(name="kv-handover-8b", op="kv", bits=8, kv_heads=8, head_dim=128, past=16000,
             tokens=77, first=0),
        # a decode step of the 4B class before its attention, float caches
        dict(name="rope-step-4b", op="rope", bits=32, pairs="halves", heads=32, kv_heads=8,
             head_dim=128, past=2047, tokens=1),
        # eight drafted tokens on the smallest model's heads of 48
        dict(name="rope-tiny-8", op="rope", bits=8, pairs="adjacent", heads=6, kv_heads=6,
             head_dim=48, past=29, tokens=8),
        # a long prompt of the 27B class into the 4-bit cache
        dict(name="rope-prompt-27b", op="rope", bits=4, pairs="halves", heads=32, kv_heads=16,
             head_dim=128, past=0, tokens=1024),
        # the smallest model's step: bound by launches
        dict(name="attn-tiny-1", op="attn", bits=8, heads=6, kv_heads=6, head_dim=48, past=33,
             tokens=1),
        # one answer token of the 8B class
        dict(name="attn-8b-1", op="attn", bits=4, heads=32, kv_heads=8, head_dim=128, past=4096,
             tokens=1),
        # one answer token on a very long document
        dict(name="attn-4b-1-long", op="attn", bits=4, heads=32, kv_heads=8, head_dim=128,
             past=131070, tokens=1),
        # speculative decoding: eight drafted tokens of the 27B class verified in one pass
        dict(name="attn-27b-8", op="attn", bits=4, heads=32, kv_heads=16, head_dim=128, past=8192,
             tokens=8),
        # a prompt on an empty cache
        dict(name="attn-4b-prompt", op="attn", bits=8, heads=32, kv_heads=8, head_dim=128, past=0,
             tokens=1024),
        # the next turn of a long conversation, a ragged number of tokens
        dict(name="attn-8b-turn", op="attn", bits=4, heads=32, kv_heads=8, head_dim=128, past=8000,
             tokens=777),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["kv", "rope", "attn", "attn"])
    kv = rng.choice([1, 2, 4, 6, 8, 16])
    hd = rng.choice([40, 48, 64, 96, 128, 128, 256])
    bits = rng.choice([4, 4, 8])
    tokens = rng.choice([1, rng.randint(2, 8), _log_int(rng, 9, 1000)])
    if op == "kv":
        past = _log_int(rng, 1, min(16000, (16 << 20) // (kv * hd) - tokens))
        return dict(op=op, bits=bits, kv_heads=kv, head_dim=hd, past=past, tokens=tokens,
                    first=rng.choice([past, rng.randint(0, past)]))
    heads = kv * rng.choice([1, 2, 4] if kv > 8 else [1, 2, 4, 5, 8])
    if op == "rope":
        return dict(op=op, bits=rng.choice([bits, 32]), pairs=rng.choice(["halves", "adjacent"]),
                    heads=heads, kv_heads=kv, head_dim=hd, past=_log_int(rng, 1, 4000),
                    tokens=tokens)
    # (the largest listed case has 777 tokens on 8000 positions of 32 heads of 128)
    most = min(130000, int(2.5e10 / (tokens * heads * hd)), (130 << 20) // (kv * hd))
    return dict(op=op, bits=bits, heads=heads, kv_heads=kv, head_dim=hd,
                past=_log_int(rng, 1, max(most, 2)), tokens=tokens)


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _keys_values(seed, n, kv_heads, hd):
    """[n][kv_heads hd] keys and values of the positions 0 .. n - 1."""
    g = _gen(2 * seed + 1)
    w = kv_heads * hd
    gain = torch.exp(0.5 * _randn(g, w))
    gain[torch.randint(0, w, (max(1, w // 64),), generator=g, device="cuda")] *= 4.0
    return _randn(g, n, w) * gain, 0.5 * _randn(g, n, w)


def _tables(n, hd):
    ex = BASE ** (-2.0 * torch.arange(hd // 2, dtype=torch.float64) / hd)
    th = torch.arange(n, dtype=torch.float64)[:, None] * ex
    return th.cos().float().cuda(), th.sin().float().cuda()


def _quads(v):
    """Rows of a float value cache in the device's order: four positions of a column side by side."""
    n, w = v.shape
    pad = torch.zeros((-n) % 4, w, dtype=v.dtype, device=v.device)
    return torch.cat([v, pad]).reshape(-1, 4, w).transpose(1, 2).contiguous()


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


def _copies(size):
    return max(1, min(16, ROTATE // max(size, 1)))


def _row_bytes(bits, hd):
    """One position of a kv head, keys and values."""
    return 2 * (hd * 4 if bits == 32 else hd * bits // 8 + -(-hd // 32))


def _fill(s, case, k, v):
    """The state's caches, rows 0 .. n - 1 in them."""
    bits, kvh, hd = case["bits"], case["kv_heads"], case["head_dim"]
    n = s.n_ctx
    copies = _copies(_row_bytes(bits, hd) * kvh * n)
    if not own:
        one = _quantise(k, kvh, hd, bits) + _quantise(v, kvh, hd, bits)
        s.caches = [tuple(t.clone() for t in one) for _ in range(copies)]
        return
    size = s.gpu.kvq_bytes(bits, n, kvh, hd)
    cache = _Dev(torch.zeros(size, dtype=torch.uint8, device="cuda"))
    zero = _Dev(torch.zeros(1, dtype=torch.int32, device="cuda"))
    k, v = _Dev(k), _Dev(v)
    torch.cuda.synchronize()
    s.gpu.kvq_write(bits, cache, n, kvh, hd, zero, n, k, v)
    s.gpu.sync()
    s.caches = [cache] + [_Dev(cache.t.clone()) for _ in range(copies - 1)]


def prepare(case, seed):
    s = SimpleNamespace(case=case, turn=0, own=own)
    if own:
        s.gpu = _gpu()
    op, kvh, hd, past, M = (case[x] for x in ("op", "kv_heads", "head_dim", "past", "tokens"))
    s.n_ctx = n = past + M
    k, v = _keys_values(seed, n, kvh, hd)
    g = _gen(2 * seed)
    s.pos = _Dev(torch.tensor([past], dtype=torch.int32, device="cuda"))
    if op != "attn":
        s.k, s.v = _Dev(k[past:].clone()), _Dev(v[past:].clone())
        k[past:], v[past:] = 0.0, 0.0
    if op != "kv":
        s.q = _Dev(1.5 * _randn(g, M, case["heads"] * hd))
        s.out = _Dev(torch.zeros_like(s.q.t))
    if op == "rope":
        s.qn, s.kn = (_Dev(1.0 + 0.1 * _randn(g, hd)) for _ in range(2))
        s.cos, s.sin = (_Dev(t) for t in _tables(n, hd))
    if case["bits"] == 32:
        s.caches = [(_Dev(k.clone()), _Dev(_quads(v)))
                    for _ in range(_copies(8 * k.numel()))]
    else:
        _fill(s, case, k, v)
    if op != "attn" and case["bits"] != 32:
        rows = n - case.get("first", past)
        s.ko, s.vo = (_Dev(torch.zeros(rows, kvh * hd, device="cuda")) for _ in range(2))
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------ the operators

def run(s):
    s.turn += 1
    return (_run_own if s.own else _run_plain)(s, s.caches[s.turn % len(s.caches)])


def _run_own(s, cache):
    c = s.case
    bits, kvh, hd, past, M, n = c["bits"], c["kv_heads"], c["head_dim"], c["past"], c["tokens"], s.n_ctx
    if c["op"] == "attn":
        s.gpu.kvq_attention(s.out, s.q, bits, cache, c["heads"], kvh, hd, M, s.pos, n)
        return s.out.t
    if c["op"] == "kv":
        s.gpu.kvq_write(bits, cache, n, kvh, hd, s.pos, M, s.k, s.v)
        s.gpu.kvq_read(bits, cache, n, kvh, hd, c["first"], n - c["first"], s.ko, s.vo)
        return [s.ko.t, s.vo.t]
    halves = c["pairs"] == "halves"
    if bits == 32:
        s.gpu.norm_rope_store(s.q, s.k, s.v, s.out, c["heads"], kvh, hd, M, s.qn, s.kn, EPS, halves,
                              s.cos, s.sin, s.pos, n, cache[0], cache[1])
        return [s.out.t, cache[0].t, cache[1].t]
    s.gpu.kvq_norm_rope_store(s.q, s.k, s.v, s.out, c["heads"], kvh, hd, M, s.qn, s.kn, EPS, halves,
                              s.cos, s.sin, s.pos, bits, cache, n)
    s.gpu.kvq_read(bits, cache, n, kvh, hd, past, M, s.ko, s.vo)
    return [s.out.t, s.ko.t, s.vo.t]


def _scales(bits):
    """Every scale in order: 3 mantissa bits, the lowest exponent's without a leading one."""
    e, m = torch.meshgrid(torch.arange(32), torch.arange(8), indexing="ij")
    d = torch.where(e == 0, m, m + 8).double() * 2.0 ** (e.clamp(min=1).double() - 20.0)
    d = d.reshape(-1)
    return d[d <= CAP[bits]]


_tables_of = {}


def _quantise(x, kvh, hd, bits):
    """Codes [n][kvh][groups][32] (int8) and scales [n][kvh][groups] (float16) of rows x.
    In 64 bits: a quotient next to a half decides a code."""
    if bits not in _tables_of:
        _tables_of[bits] = _scales(bits).cuda()
    table, h = _tables_of[bits], HALF[bits]
    n, ng = x.shape[0], -(-hd // 32)
    codes = torch.empty(n, kvh, ng, 32, dtype=torch.int8, device=x.device)
    scales = torch.empty(n, kvh, ng, dtype=torch.float16, device=x.device)
    for i in range(0, n, 8192):
        g = x[i:i + 8192].double().reshape(-1, kvh, hd)
        g = torch.nn.functional.pad(g, (0, 32 * ng - hd)).reshape(-1, kvh, ng, 32)
        lim = torch.maximum(g.amax(-1) / (h - 0.5), -g.amin(-1) / (h + 0.5)).clamp(min=0.0)
        d = table[torch.searchsorted(table, lim).clamp(max=len(table) - 1)]
        r = torch.where(d[..., None] > 0, g / d[..., None], torch.zeros_like(g))
        codes[i:i + 8192] = torch.round(r).clamp(-h, h - 1).to(torch.int8)
        scales[i:i + 8192] = d.to(torch.float16)
    return codes, scales


def _values(codes, scales, hd):
    """[n][kvh][hd] floats of a cache's rows."""
    x = codes.float() * scales.float()[..., None]
    return x.flatten(2)[..., :hd]


def _norm_rope(x, heads, hd, w, cos, sin, pairs):
    """In 64 bits: the result's code depends on its last bits."""
    x = x.double().reshape(-1, heads, hd)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
    c, s = cos.double()[:, None, :], sin.double()[:, None, :]
    a, b = (x[..., :hd // 2], x[..., hd // 2:]) if pairs == "halves" else (x[..., ::2], x[..., 1::2])
    ra, rb = a * c - b * s, a * s + b * c
    y = torch.cat([ra, rb], -1) if pairs == "halves" else torch.stack([ra, rb], -1).flatten(-2)
    return y.flatten(1).float()


def _run_plain(s, cache):
    c = s.case
    bits, kvh, hd, past, M, n = c["bits"], c["kv_heads"], c["head_dim"], c["past"], c["tokens"], s.n_ctx
    if c["op"] == "attn":
        kc, ks, vc, vs = cache
        heads, g = c["heads"], c["heads"] // kvh
        k = _values(kc, ks, hd).permute(1, 2, 0).contiguous()      # [kvh][hd][n]
        v = _values(vc, vs, hd).permute(1, 0, 2).contiguous()      # [kvh][n][hd]
        q = s.q.t.reshape(M, kvh, g, hd).permute(1, 0, 2, 3).reshape(kvh, M * g, hd)
        sc = torch.matmul(q.contiguous(), k) * (1.0 / math.sqrt(hd))
        last = past + torch.arange(M, device=sc.device)
        hidden = torch.arange(n, device=sc.device)[None, :] > last[:, None]
        sc = sc.reshape(kvh, M, g, n).masked_fill_(hidden[:, None, :], -math.inf)
        e = torch.exp(sc - sc.amax(-1, keepdim=True))
        o = torch.matmul(e.reshape(kvh, M * g, n), v) / e.sum(-1).reshape(kvh, M * g, 1)
        s.out.t.copy_(o.reshape(kvh, M, g, hd).permute(1, 0, 2, 3).reshape(M, heads * hd))
        return s.out.t
    k, v = s.k.t, s.v.t
    if c["op"] == "rope":
        cos, sin = s.cos.t[past:n], s.sin.t[past:n]
        s.out.t.copy_(_norm_rope(s.q.t, c["heads"], hd, s.qn.t, cos, sin, c["pairs"]))
        k = _norm_rope(k, kvh, hd, s.kn.t, cos, sin, c["pairs"])
        if bits == 32:
            p = torch.arange(past, n, device=k.device)
            cache[0].t[past:n] = k
            cache[1].t[p // 4, :, p % 4] = v
            return [s.out.t, cache[0].t, cache[1].t]
    for i, x in ((0, k), (2, v)):
        codes, scales = _quantise(x, kvh, hd, bits)
        cache[i][past:n] = codes
        cache[i + 1][past:n] = scales
    first = c.get("first", past)
    s.ko.t.copy_(_values(cache[0][first:n], cache[1][first:n], hd).flatten(1))
    s.vo.t.copy_(_values(cache[2][first:n], cache[3][first:n], hd).flatten(1))
    return [s.ko.t, s.vo.t] if c["op"] == "kv" else [s.out.t, s.ko.t, s.vo.t]


# ------------------------------------------------------------ what it takes

def work(case):
    bits, kvh, hd, past, M = (case[x] for x in ("bits", "kv_heads", "head_dim", "past", "tokens"))
    row = _row_bytes(bits, hd) * kvh
    flat = 8 * kvh * hd
    if case["op"] == "attn":
        pairs = M * past + M * (M + 1) // 2
        return {"bytes": (past + M) * row + 8 * M * case["heads"] * hd,
                "flops": 4 * pairs * case["heads"] * hd}
    if case["op"] == "kv":
        n = past + M - case["first"]
        return {"bytes": M * (flat + row) + n * (flat + row), "flops": 2 * (M + n) * 2 * kvh * hd}
    q = 8 * case["heads"] * hd
    back = 0 if bits == 32 else flat + row
    return {"bytes": M * (q + flat + row + back), "flops": 8 * M * (case["heads"] + kvh) * hd}


# ------------------------------------------------------------- in 64 bits

def _held(x, bits):
    """The values, in 64 bits, that a cache holds for groups x [..., up to 32]."""
    h = HALF[bits]
    hi, lo = x.max(-1, keepdim=True).values, x.min(-1, keepdim=True).values
    need = torch.maximum(hi / (h - 0.5), lo / -(h + 0.5)).clamp(min=0.0)
    e = torch.frexp(need.clamp(min=2.0 ** -16)).exponent.long()     # need < 2^e
    step = ((e - 4 + 1023) << 52).view(torch.float64)               # 2^(e - 4), bit by bit
    d = (torch.ceil(need / step) * step).clamp(max=CAP[bits])
    t = x / torch.where(d > 0, d, torch.ones_like(d))
    r = torch.floor(t)
    f = t - r
    r = r + ((f > 0.5) | ((f == 0.5) & (r % 2 != 0))).double()
    return r.clamp(-h, h - 1) * d


def _held_rows(x, kvh, hd, bits):
    """[n][kvh hd] rows as a cache gives them back."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for h in range(kvh):
        for d in range(h * hd, (h + 1) * hd, 32):
            e = min(d + 32, (h + 1) * hd)
            out[:, d:e] = _held(x[:, d:e].double(), bits)
    return out


def _turned(x, hd, w, n0, pairs):
    """One head's rows x at positions n0 .., normed and rotated by the float tables, in 64 bits."""
    x = x.double()
    x = x * w.double() / (x.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt()
    cos, sin = (t[n0:].double() for t in _tables(n0 + x.shape[0], hd))
    y = torch.empty_like(x)
    for j in range(hd // 2):
        a, b = (j, j + hd // 2) if pairs == "halves" else (2 * j, 2 * j + 1)
        y[:, a] = x[:, a] * cos[:, j] - x[:, b] * sin[:, j]
        y[:, b] = x[:, a] * sin[:, j] + x[:, b] * cos[:, j]
    return y


def exact(case, seed):
    op, kvh, hd, past, M = (case[x] for x in ("op", "kv_heads", "head_dim", "past", "tokens"))
    bits, n = case["bits"], past + M
    k, v = _keys_values(seed, n, kvh, hd)
    g = _gen(2 * seed)
    if op == "attn":
        heads = case["heads"]
        q = (1.5 * _randn(g, M, heads * hd)).double()
        k, v = (_held_rows(x, kvh, hd, bits) for x in (k, v))
        out = torch.empty(M, heads * hd, dtype=torch.float64, device="cuda")
        seen = torch.arange(n, device="cuda")[None, :] <= past + torch.arange(M, device="cuda")[:, None]
        for h in range(heads):
            at, kv = slice(h * hd, (h + 1) * hd), slice(h // (heads // kvh) * hd, (h // (heads // kvh) + 1) * hd)
            p = torch.matmul(q[:, at], k[:, kv].t().contiguous()) / math.sqrt(hd)
            p = torch.softmax(torch.where(seen, p, torch.full_like(p, -math.inf)), -1)
            out[:, at] = torch.matmul(p, v[:, kv].contiguous())
        return out
    if op == "kv":
        first = case["first"]
        return [_held_rows(x[first:], kvh, hd, bits) for x in (k, v)]
    heads = case["heads"]
    q = 1.5 * _randn(g, M, heads * hd)
    qn, kn = (1.0 + 0.1 * _randn(g, hd) for _ in range(2))
    pairs = case["pairs"]
    qo, ko = (torch.cat([_turned(x[:, h * hd:(h + 1) * hd], hd, w, past, pairs) for h in range(nh)], 1)
              for x, nh, w in ((q, heads, qn), (k[past:], kvh, kn)))
    if bits != 32:
        # (a key is rounded to a float before it is quantised)
        return [qo, _held_rows(ko.float(), kvh, hd, bits), _held_rows(v[past:], kvh, hd, bits)]
    k = k.double()
    k[past:] = ko
    return [qo, k, _quads(v.double())]
