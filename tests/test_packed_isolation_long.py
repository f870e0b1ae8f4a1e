"""Packed sequences long enough for two tiles per thread block (head_dim up to 128): nothing of a neighbour's rows, or of rows that are
nobody's, reaches a result, and nothing outside the sequences is written.  That form zeroes the rows of V behind a sequence in a
buffer that both tiles read, and stores cut tiles of its own."""
import pytest
import torch

pytestmark = pytest.mark.gpu

LONG = {64: 8192, 128: 4096}      # keys per sequence on average from which it is taken, with 256 queries or more


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _starts(lens):
    return torch.tensor([0] + lens).cumsum(0).int().cuda()


def _rows(T, heads, D, dtype, seed):
    return torch.randn(T, heads, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def _long(D, lens_q, lens_k):
    return sum(lens_k) >= LONG[D] * len(lens_k) and sum(lens_q) >= 256 * len(lens_q)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_between_rows_that_are_not_finite(D, causal, dtype):
    from acctransformer_b200 import _lib, flash_attention_packed
    N, gap = 2, 50
    # queries: a last pair with one tile that is cut, and with two; keys: last tiles that are cut, by one row and by nearly all
    lens_q, lens_k = [1100, 401], [3 * LONG[D] + 127, 2 * LONG[D] + 385]
    q, k, v = _rows(sum(lens_q), N, D, dtype, 1), _rows(sum(lens_k), 1, D, dtype, 2), _rows(sum(lens_k), 1, D, dtype, 3)
    assert _long(D, lens_q, lens_k)
    want, sums = flash_attention_packed(q, k, v, _starts(lens_q), _starts(lens_k), causal=causal, return_lse=True)
    assert want.isfinite().all() and sums.isfinite().all()
    lq, lk = [gap, lens_q[0], gap, lens_q[1], gap], [gap, lens_k[0], gap, lens_k[1], gap]
    assert _long(D, lq, lk)
    for bad in (float("nan"), float("inf"), torch.finfo(dtype).min):
        def spread(x, lens):
            none = torch.full((gap,) + x.shape[1:], bad, device="cuda", dtype=dtype)
            return torch.cat([none, x[:lens[0]], none, x[lens[0]:], none])
        y, lse = flash_attention_packed(spread(q, lens_q), spread(k, lens_k), spread(v, lens_k), _starts(lq), _starts(lk), causal=causal, return_lse=True)
        at = [slice(gap, gap + lens_q[0]), slice(2 * gap + lens_q[0], 2 * gap + sum(lens_q))]
        assert torch.equal(torch.cat([y[i] for i in at]), want) and torch.equal(torch.cat([lse[:, i] for i in at], 1), sums)
    torch.cuda.synchronize()
    _lib.device_status()


@pytest.mark.parametrize("D", [64, 128])
def test_rows_outside_are_not_written(D):
    from acctransformer_b200 import flash_attention_packed
    N, dtype = 2, torch.float16
    lens_q, lens_k = [300, 785, 300], [LONG[D], 2 * LONG[D] + 1, LONG[D]]
    q, k, v = _rows(sum(lens_q), N, D, dtype, 4), _rows(sum(lens_k), 1, D, dtype, 5), _rows(sum(lens_k), 1, D, dtype, 6)
    cu_q, cu_k = _starts(lens_q), _starts(lens_k)
    assert _long(D, lens_q, lens_k)
    want = flash_attention_packed(q, k, v, cu_q, cu_k)
    out = torch.full_like(q, 7.0)
    flash_attention_packed(q, k, v, cu_q[1:3], cu_k[1:3], out=out)
    assert torch.equal(out[300:1085], want[300:1085]) and (out[:300] == 7).all() and (out[1085:] == 7).all()
