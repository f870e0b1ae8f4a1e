"""Eviction reads one cache and writes another: memory that is in both is refused, other pages of one pool are not."""
import ctypes as C

import pytest
import torch

from acctransformer_b200 import _lib, build as _build

A = 0x1000000      # some aligned address: nothing that is refused looks at it
SHAPE = 2
RECORD = 1280      # of 16 rows of one head of 64


@pytest.fixture(scope="module")
def lib():
    _build.build()
    return _lib.load()


def _cache(records, table=None, **kw):
    c = _lib.Kv4CacheArgs()
    c.dtype, c.B, c.N_kv, c.S_max, c.D, c.records, c.block_table = _lib.ACCT_F16, 2, 2, 100, 64, records, table
    if table is not None:
        c.page_size, c.max_pages, c.num_pages = 32, 4, 10
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _evict(**kw):
    a = _lib.Kv4EvictArgs()
    a.weights, a.seq_lens, a.keep, a.recent, a.weights_out, a.kept, a.seq_lens_out = A, A, 8, 2, 2 * A, 4 * A, 2 * A
    for k, v in kw.items():
        setattr(a, k, v)
    return a


HELD = 2 * 2 * 7 * RECORD             # bytes of a contiguous cache of 100 slots
POOL = 10 * 2 * 2 * RECORD            # of the pool


@pytest.mark.parametrize("src, dst", [
    ((A,), (A,)), ((A,), (A + 16,)), ((A,), (A + HELD - 16,)), ((A + HELD - 16,), (A,)), ((A,), (A - 16,)),
    ((A, 8 * A), (A, 8 * A)), ((A, 8 * A), (A,)), ((A,), (A, 8 * A)), ((A, 8 * A), (A + POOL - 16,)), ((A + POOL - 16,), (A, 8 * A)),
    ((A, 8 * A), (A + 2 * RECORD, 9 * A)), ((A + POOL - 16, 8 * A), (A, 9 * A)),
], ids=str)
def test_records_in_both(lib, src, dst):
    assert lib.acct_kv4_evict(_cache(*src), _cache(*dst), _evict(), None) == SHAPE
    assert b"in place" in lib.acct_last_error()


def test_a_small_cache_inside_a_large_one(lib):
    assert lib.acct_kv4_evict(_cache(A, S_max=2000), _cache(A + 100 * RECORD, S_max=8), _evict(), None) == SHAPE
    assert lib.acct_kv4_evict(_cache(A + 100 * RECORD, S_max=8), _cache(A, S_max=2000), _evict(keep=8), None) == SHAPE


@pytest.mark.parametrize("kw", [{"weights_out": A}, {"weights_out": A + 4}, {"weights_out": A + 1596}, {"weights_out": A - 1596}, {"seq_lens_out": A},
                                {"seq_lens_out": A + 4}, {"seq_lens_out": A - 4}], ids=str)
def test_weights_and_lengths_in_both(lib, kw):
    assert lib.acct_kv4_evict(_cache(A), _cache(2 * A), _evict(**kw), None) == SHAPE
    assert b"in place" in lib.acct_last_error()


@pytest.mark.gpu
def test_into_other_pages_of_the_same_pool():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from acctransformer_b200 import Kv4Cache
    B, N_kv, S, D, page, dtype = 2, 2, 128, 64, 16, torch.float16
    pages = torch.randperm(2 * B * S // page).int().cuda()
    first, second = pages.view(2, B, -1).contiguous()
    pool = Kv4Cache(B, N_kv, S, D, dtype=dtype, page_size=page, block_table=first, num_pages=len(pages))
    apart = Kv4Cache(B, N_kv, S, D, dtype=dtype)
    k, v = (torch.randn(B * S, N_kv, D, device="cuda").to(dtype) for _ in range(2))
    zero, cu = torch.zeros(B, dtype=torch.int32, device="cuda"), torch.tensor([0, S, 2 * S], dtype=torch.int32, device="cuda")
    pool.append(k, v, zero, cu)
    w, lens = torch.rand(B, N_kv, S, device="cuda"), torch.tensor([S, 77], dtype=torch.int32, device="cuda")
    want = pool.evict(w, lens, 60, 9, apart)

    c = [_lib.Kv4CacheArgs() for _ in range(2)]
    for x, table in zip(c, (first, second)):
        x.dtype, x.B, x.N_kv, x.S_max, x.D, x.records, x.block_table = _lib.ACCT_F16, B, N_kv, S, D, pool.records.data_ptr(), table.data_ptr()
        x.page_size, x.max_pages, x.num_pages = page, S // page, len(pages)
    got = [torch.empty_like(x) for x in want]
    a = _lib.Kv4EvictArgs()
    a.weights, a.seq_lens, a.keep, a.recent = w.data_ptr(), lens.data_ptr(), 60, 9
    a.kept, a.weights_out, a.seq_lens_out = (x.data_ptr() for x in got)
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    _lib.check(_lib.load().acct_kv4_evict(c[0], c[1], a, stream))
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    first.copy_(second)                                      # the pool as the smaller cache
    cu = torch.tensor([0, 60, 120], dtype=torch.int32, device="cuda")
    for x, y in zip(pool.read(zero, cu, total=120), apart.read(zero, cu, total=120)):
        assert torch.equal(x, y)
