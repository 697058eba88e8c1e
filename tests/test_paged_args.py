"""Refusals of the paged caches' entry points: every bad call returns its status before anything
touches a device, so they run here over a context that is only memory."""
import ctypes as C

import pytest

import rustfox_amd as rf

ARG, UNSUPPORTED = 1, 5
CTX = C.create_string_buffer(4096)
BUF = (C.c_char * (1 << 12 + 16))()
P = (C.addressof(BUF) + 15) // 16 * 16
CACHE = dict(type=rf.F16, k=P, v=P, n_pages=40, page_size=16, n_head_kv=2, head_dim=64, table=P, n_seqs=3,
             max_pages=10, weight=P, position=P)
FREQ = dict(base=1e4, scale=1.0, ext=0.0, beta_fast=32.0, beta_slow=1.0, orig_ctx=0.0, magnitude=1.0,
            factors=None)
BAD_CACHES = [(dict(type=0), UNSUPPORTED), (dict(type=4), UNSUPPORTED), (dict(k=None), ARG), (dict(v=None), ARG),
              (dict(table=None), ARG), (dict(n_pages=0), ARG), (dict(page_size=0), ARG), (dict(n_head_kv=0), ARG),
              (dict(head_dim=0), ARG), (dict(n_seqs=0), ARG), (dict(max_pages=0), ARG),
              (dict(head_dim=68), UNSUPPORTED), (dict(head_dim=264), UNSUPPORTED), (dict(page_size=8), UNSUPPORTED),
              (dict(page_size=48), UNSUPPORTED), (dict(page_size=8192), UNSUPPORTED), (dict(k=P + 8), ARG),
              (dict(v=P + 2), ARG), (dict(n_pages=(1 << 31) + 1), ARG), (dict(n_seqs=65536), ARG),
              (dict(n_head_kv=4097), ARG), (dict(n_seqs=1024, n_head_kv=1025), ARG),
              (dict(max_pages=(1 << 26) + 1), ARG), (dict(max_pages=2 ** 64 - 1), ARG), (dict(weight=None), ARG),
              (dict(position=None), ARG), (dict(weight=P + 4), ARG), (dict(position=P + 8), ARG)]

STORE = dict(ctx=C.addressof(CTX), cache=CACHE, q=P, qs=256, o=P, os=256, nh=4, k=P, ks=128, v=P, vs=128, M=3,
             qn=P, kn=P, eps=1e-6, pairs=0, n_rot=64, cos=P, sin=P, n_table=100, pos=P, seq=None, row=None)
ATTN = dict(ctx=C.addressof(CTX), cache=CACHE, o=P, os=256, q=P, qs=256, nh=4, M=3, length=P, seq=None, weigh=1)
EVICT = dict(ctx=C.addressof(CTX), cache=CACHE, length=P, kept=P + 64, keep=20, recent=5)
TABLES = dict(ctx=C.addressof(CTX), cos=P, sin=P, p0=0, n=100, n_rot=64, freq=FREQ)
NONE = dict(weight=None, position=None)
INF, NAN = float("inf"), float("nan")

CALLS = {
    "store": ("fox_gpu_paged_rope_store", STORE, [
        (dict(ctx=None), ARG), (dict(cache=None), ARG), (dict(q=None), ARG), (dict(o=None), ARG), (dict(k=None), ARG),
        (dict(v=None), ARG), (dict(cos=None), ARG), (dict(sin=None), ARG), (dict(pos=None), ARG), (dict(nh=0), ARG),
        (dict(M=0), ARG), (dict(n_table=0), ARG), (dict(n_table=(1 << 30) + 1), ARG), (dict(pairs=2), ARG),
        (dict(n_rot=0), ARG), (dict(n_rot=63), ARG), (dict(n_rot=66), ARG), (dict(M=4), ARG),
        (dict(M=1025, seq=P), ARG), (dict(nh=65536, qs=1 << 23, os=1 << 23), ARG), (dict(qs=255), ARG),
        (dict(os=255), ARG), (dict(ks=127), ARG), (dict(vs=127), ARG)]),
    "attention": ("fox_gpu_paged_attention", ATTN, [
        (dict(ctx=None), ARG), (dict(cache=None), ARG), (dict(o=None), ARG), (dict(q=None), ARG),
        (dict(length=None), ARG), (dict(nh=0), ARG), (dict(nh=5), ARG), (dict(nh=65538, qs=1 << 23, os=1 << 23), ARG),
        (dict(M=0), ARG), (dict(M=4), ARG), (dict(M=1025, seq=P, weigh=0), ARG), (dict(qs=255), ARG),
        (dict(os=255), ARG), (dict(seq=P), ARG), (dict(cache=dict(CACHE, **NONE)), ARG)]),
    "evict": ("fox_gpu_paged_evict", EVICT, [
        (dict(ctx=None), ARG), (dict(cache=None), ARG), (dict(length=None), ARG), (dict(kept=None), ARG),
        (dict(keep=0), ARG), (dict(recent=21), ARG), (dict(kept=P), ARG), (dict(kept=P + 8), ARG),
        (dict(length=P + 8, kept=P), ARG), (dict(cache=dict(CACHE, **NONE)), ARG)]),
    "tables": ("fox_gpu_rope_tables", TABLES, [
        (dict(ctx=None), ARG), (dict(cos=None), ARG), (dict(sin=None), ARG), (dict(freq=None), ARG), (dict(n=0), ARG),
        (dict(n_rot=0), ARG), (dict(n_rot=63), UNSUPPORTED), (dict(n_rot=258), UNSUPPORTED),
        (dict(n=(1 << 30) + 1), ARG), (dict(p0=(1 << 30) + 1), ARG), (dict(p0=1 << 30, n=1), ARG),
        (dict(p0=2 ** 64 - 1, n=2), ARG), (dict(n=1 << 30, n_rot=256), ARG)] +
        [(dict(freq=dict(FREQ, **f)), ARG) for f in (
            dict(base=0.0), dict(base=-1.0), dict(base=NAN), dict(base=INF), dict(scale=NAN), dict(scale=INF),
            dict(ext=NAN), dict(magnitude=INF), dict(ext=1.0), dict(ext=1.0, orig_ctx=64.0, base=1.0),
            dict(ext=1.0, orig_ctx=64.0, beta_fast=0.0), dict(ext=1.0, orig_ctx=64.0, beta_slow=-1.0),
            dict(ext=1.0, orig_ctx=NAN), dict(ext=1.0, orig_ctx=INF))]),
}


def call(lib, fn, args):
    got = []
    for name, v in args.items():
        if name == "cache" and v is not None:
            v = C.byref(rf.Paged(*v.values()))
        if name == "freq" and v is not None:
            v = C.byref(rf.RopeFreq(*v.values()))
        got.append(v)
    return getattr(lib, fn)(*got)


@pytest.mark.parametrize("name", list(CALLS))
def test_refusals(name):
    lib = rf.gpu_lib()
    fn, base, bad = CALLS[name]
    if "cache" in base:
        bad = bad + [(dict(cache=dict(CACHE, **c)), want) for c, want in BAD_CACHES]
    for change, want in bad:
        got = call(lib, fn, dict(base, **change))
        assert got == want, (change, got, lib.fox_gpu_last_error())
        assert lib.fox_gpu_last_error(), change
