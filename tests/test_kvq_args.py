"""Refusals of the quantised-cache entry points: every bad call returns its status before
anything touches a device, so they run here over a context that is only memory."""
import ctypes as C

import pytest

import rustfox_amd as rf

ARG, UNSUPPORTED = 1, 5
CTX = C.create_string_buffer(4096)
BUF = (C.c_char * (1 << 12 + 16))()
P = (C.addressof(BUF) + 15) // 16 * 16


@pytest.fixture(scope="module")
def lib():
    return rf.gpu_lib()


def test_bytes(lib):
    size = lib.fox_gpu_kvq_bytes
    # 32 positions of one head: codes of keys and values, a scale byte per 32 of them
    assert size(rf.KV_Q4, 32, 1, 128) == 2 * (32 * 64 + 32 * 4)
    assert size(rf.KV_Q8, 1, 1, 128) == 2 * (32 * 128 + 32 * 4)
    assert size(rf.KV_Q4, 33, 3, 48) == 3 * 2 * 2 * (32 * 32 + 32 * 2)
    assert size(rf.KV_Q4, 1 << 30, 32767, 256) == 32767 * (1 << 25) * 2 * (32 * 128 + 32 * 8)
    for hd, width in [(2, 32), (32, 32), (34, 64), (80, 96), (130, 192), (194, 256), (256, 256)]:
        assert size(rf.KV_Q8, 32, 1, hd) == 2 * (32 * width + width), hd
    for bad in [(5, 32, 1, 128), (4, 0, 1, 128), (4, 32, 0, 128), (4, 32, 1, 0), (4, 32, 1, 258),
                (4, 32, 1, 7), (4, (1 << 30) + 1, 1, 128), (4, 32, 32768, 128)]:
        assert size(*bad) == 0, bad


WRITE = dict(ctx=C.addressof(CTX), kv=4, cache=P, n_ctx=100, nkv=2, hd=64, pos=P, M=3, k=P, ks=128,
             v=P, vs=128)
READ = dict(ctx=C.addressof(CTX), kv=4, cache=P, n_ctx=100, nkv=2, hd=64, p0=1, n=3, k=P, ks=128,
            v=P, vs=128)
ROPE = dict(ctx=C.addressof(CTX), q=P, qs=256, o=P, os=256, k=P, ks=128, v=P, vs=128, nh=4, nkv=2,
            hd=64, M=3, qn=P, kn=P, eps=1e-6, pairs=0, cos=P, sin=P, pos=P)
ROPE_F = dict(ROPE, n_ctx=100, kc=P, vc=P)
ROPE_Q = dict(ROPE, kv=8, cache=P, n_ctx=100)
ATTN = dict(ctx=C.addressof(CTX), o=P, os=256, q=P, qs=256, kv=4, cache=P, nh=4, nkv=2, hd=64, M=3,
            pos=P, n_ctx=100)
SHAPE = [(dict(n_ctx=0), ARG), (dict(nkv=0), ARG), (dict(hd=0), ARG), (dict(kv=3), UNSUPPORTED),
         (dict(hd=63), UNSUPPORTED), (dict(hd=258), UNSUPPORTED), (dict(n_ctx=(1 << 30) + 1), ARG)]

CALLS = {
    "write": ("fox_gpu_kvq_write", WRITE, SHAPE + [
        (dict(ctx=None), ARG), (dict(cache=None), ARG), (dict(pos=None), ARG), (dict(k=None), ARG),
        (dict(v=None), ARG), (dict(M=0), ARG), (dict(M=101), ARG), (dict(ks=127), ARG),
        (dict(vs=127), ARG), (dict(cache=P + 8), ARG), (dict(nkv=32768, ks=1 << 22, vs=1 << 22), ARG),
        (dict(n_ctx=1 << 30, M=(1 << 28) + 1), ARG)]),
    "read": ("fox_gpu_kvq_read", READ, SHAPE + [
        (dict(ctx=None), ARG), (dict(cache=None), ARG), (dict(k=None, v=None), ARG), (dict(n=0), ARG),
        (dict(p0=98), ARG), (dict(p0=100), ARG), (dict(n=101), ARG), (dict(n=2 ** 64 - 1), ARG),
        (dict(ks=127), ARG), (dict(vs=127), ARG), (dict(cache=P + 4), ARG),
        (dict(n_ctx=1 << 30, n=(1 << 28) + 1), ARG)]),
    "rope": ("fox_gpu_norm_rope_store", ROPE_F, [s for s in SHAPE if "kv" not in s[0]] + [
        (dict(ctx=None), ARG), (dict(q=None), ARG), (dict(o=None), ARG), (dict(k=None), ARG),
        (dict(v=None), ARG), (dict(cos=None), ARG), (dict(sin=None), ARG), (dict(pos=None), ARG),
        (dict(kc=None), ARG), (dict(vc=None), ARG), (dict(nh=0), ARG), (dict(M=0), ARG),
        (dict(M=1025), ARG), (dict(pairs=2), ARG), (dict(qs=255), ARG), (dict(os=255), ARG),
        (dict(ks=127), ARG), (dict(vs=127), ARG)]),
    "kvq_rope": ("fox_gpu_kvq_norm_rope_store", ROPE_Q, SHAPE + [
        (dict(ctx=None), ARG), (dict(q=None), ARG), (dict(cache=None), ARG), (dict(cache=P + 8), ARG),
        (dict(nh=0), ARG), (dict(M=0), ARG), (dict(M=1025), ARG), (dict(pairs=-1), ARG),
        (dict(nh=65533, qs=1 << 24, os=1 << 24), ARG),
        (dict(ks=127), ARG)]),
    "attention": ("fox_gpu_kvq_attention", ATTN, SHAPE + [
        (dict(ctx=None), ARG), (dict(o=None), ARG), (dict(q=None), ARG), (dict(cache=None), ARG),
        (dict(pos=None), ARG), (dict(nh=0), ARG), (dict(nh=5), ARG), (dict(M=0), ARG),
        (dict(M=1025), ARG), (dict(qs=255), ARG), (dict(os=255), ARG), (dict(cache=P + 8), ARG),
        (dict(hd=192, nkv=1, nh=65535, M=33, qs=1 << 24, os=1 << 24), ARG)]),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_refusals(lib, name):
    fn, base, bad = CALLS[name]
    for change, want in bad:
        got = getattr(lib, fn)(*dict(base, **change).values())
        assert got == want, (change, got, lib.fox_gpu_last_error())
        assert lib.fox_gpu_last_error(), change
