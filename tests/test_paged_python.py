"""The Python calls of the paged caches pass on what they are given, whether the cache is a PagedCache or a
struct: over a library that only writes its arguments down."""
import ctypes as C
from types import SimpleNamespace

import pytest

import rustfox_amd as rf


class Written:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


def array(ptr):
    return SimpleNamespace(ptr=ptr)


def caches():
    names = dict(k=0x1000, v=0x2000, table=0x3000, weight=0x4000, position=0x5000)
    a = {n: array(p) for n, p in names.items()}
    yield rf.PagedCache(rf.BF16, a["k"], a["v"], 40, 16, 2, 64, a["table"], 3, 10, a["weight"], a["position"])
    yield rf.Paged(type=rf.BF16, n_pages=40, page_size=16, n_head_kv=2, head_dim=64, n_seqs=3, max_pages=10, **names)


@pytest.mark.parametrize("cache", caches(), ids=["PagedCache", "Paged"])
def test_a_cache_and_its_struct(cache):
    gpu = rf.Gpu.__new__(rf.Gpu)
    gpu.lib, gpu.ctx = Written(), None
    q, o, n = array(0x100), array(0x200), array(0x300)
    gpu.paged_rope_store(cache, q, o, 8, q, q, 3, n, 64, 0, q, q, 100)
    gpu.paged_attention(cache, o, q, 8, 3, n, weigh=True)
    gpu.paged_evict(cache, n, o, 20, 5)
    store, attention, evict = gpu.lib.calls
    for name, args in gpu.lib.calls:
        c = C.cast(args[1], C.POINTER(rf.Paged)).contents
        assert (c.type, c.k, c.v, c.n_pages, c.page_size, c.n_head_kv, c.head_dim, c.table, c.n_seqs, c.max_pages, c.weight,
                c.position) == (30, 0x1000, 0x2000, 40, 16, 2, 64, 0x3000, 3, 10, 0x4000, 0x5000), name
    # rows' widths where no stride is given
    assert store[1][3] == store[1][5] == 8 * 64 and store[1][8] == store[1][10] == 2 * 64
    assert attention[1][3] == attention[1][5] == 8 * 64
    assert evict[1][2:] == (0x300, 0x200, 20, 5)
