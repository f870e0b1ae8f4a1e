"""Attention of packed sequences against float64, at the lengths and layouts where it can go wrong.

u = 2^-11 (float16) or 2^-8 (bfloat16): P is rounded to 16 bits for P V and the result once more, so |y - exact| <=
2 u sum_j p_j |v_j| up to the scores' own error: fp32 sums of products whose absolute values add up to A, so a probability is off
by a factor of at most exp(2 e) with e = 2^-20 A plus a few units of 2^-22 for the exponential and the sum."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _starts(lens):
    return torch.tensor([0] + lens).cumsum(0).int().cuda()


def _rows(T, heads, D, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(T, heads, D, device="cuda", generator=g).to(dtype)


def _check(q, k, v, lens_q, lens_k, y, lse=None, causal=True, scale=None, at_q=0, at_k=0):
    from acctransformer_b200 import _lib
    torch.cuda.synchronize()
    _lib.device_status()
    N, D = q.shape[1:]
    per = N // k.shape[1]
    u = UNIT[q.dtype]
    scale = D ** -0.5 if scale is None else scale
    for n, m in zip(lens_q, lens_k):
        qq = q[at_q:at_q + n].double().transpose(0, 1)
        kk, vv = (x[at_k:at_k + m].double().transpose(0, 1).repeat_interleave(per, 0) for x in (k, v))
        x = scale * qq @ kk.transpose(1, 2)
        A = float((scale * qq.abs() @ kk.abs().transpose(1, 2)).max()) if n and m else 0.0
        if causal:
            x = x.masked_fill(torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1), -math.inf)
        sums = x.logsumexp(-1) if m else torch.full((N, n), -math.inf, device="cuda", dtype=torch.float64)
        p = torch.where(sums[..., None] == -math.inf, 0.0, (x - sums[..., None]).exp())
        want, size = (p @ vv).transpose(0, 1), (p @ vv.abs()).transpose(0, 1)
        e = 2.0 ** -20 * A + 2.0 ** -18
        got = y[at_q:at_q + n].double()
        assert ((got - want).abs() <= size * (3 * u + math.expm1(2 * e)) + 1e-6 * (size > 0)).all(), (n, m, float((got - want).abs().max()))
        if lse is not None:
            mine = lse[:, at_q:at_q + n].double()
            assert torch.equal(mine == -math.inf, sums == -math.inf)
            seen = sums != -math.inf
            assert ((mine - sums)[seen].abs() <= e + 2.0 ** -22 * sums[seen].abs() + 1e-6).all()
        at_q, at_k = at_q + n, at_k + m


LENS = [
    [1], [77], [128], [129], [256], [257], [1000],
    [1, 1, 1, 1, 1], [0, 5, 0, 0, 300, 1, 0], [127, 128, 129, 255, 256, 257, 1],
    [600, 3, 2, 511, 64, 1], [40] * 40,
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(map(str, x[:7])))
@pytest.mark.parametrize("D, N, N_kv", [(128, 4, 1), (64, 3, 3), (40, 2, 1), (80, 6, 2), (160, 2, 1)])
def test_lengths(D, N, N_kv, lens, causal, dtype):
    from acctransformer_b200 import flash_attention_packed
    T = sum(lens)
    q, k, v = _rows(T, N, D, dtype, 1), _rows(T, N_kv, D, dtype, 2), _rows(T, N_kv, D, dtype, 3)
    y, lse = flash_attention_packed(q, k, v, _starts(lens), causal=causal, return_lse=True)
    assert y.shape == q.shape and y.dtype == dtype and lse.shape == (N, T)
    _check(q, k, v, lens, lens, y, lse, causal)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D, N, N_kv", [(128, 8, 2), (64, 2, 2), (256, 2, 1), (8, 1, 1)])
def test_prefixes_and_queries_that_see_nothing(D, N, N_kv, dtype):
    from acctransformer_b200 import flash_attention_packed
    #         behind a prefix            one query        fewer keys than queries: the first see none   no keys, no queries
    lens_q = [100, 256, 300, 64, 128, 1, 1, 1, 200, 300, 129, 5, 30, 0, 0]
    lens_k = [177, 300, 1000, 65, 1024, 1, 128, 700, 150, 1, 128, 0, 0, 40, 0]
    q, k, v = _rows(sum(lens_q), N, D, dtype, 4), _rows(sum(lens_k), N_kv, D, dtype, 5), _rows(sum(lens_k), N_kv, D, dtype, 6)
    for causal in (True, False):
        y, lse = flash_attention_packed(q, k, v, _starts(lens_q), _starts(lens_k), causal=causal, return_lse=True, scale=0.3)
        _check(q, k, v, lens_q, lens_k, y, lse, causal, 0.3)


# on average: just long enough for two tiles per block (4 096 keys, or 8 192 of 64), keys just too few, queries just too few, ...
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens_q, lens_k", [([256], [4096]), ([256], [4095]), ([255], [4096]), ([1, 511], [4096, 4096]), ([700, 0, 69], [5000, 1, 7300]),
                                            ([513, 300, 1], [9001, 299, 4000]), ([4229], [4229]), ([256], [8192]), ([300, 212], [10000, 6384])],
                         ids=str)
@pytest.mark.parametrize("D, N, N_kv", [(128, 4, 1), (64, 3, 3), (72, 2, 1)])
def test_long_sequences(D, N, N_kv, lens_q, lens_k, dtype):
    from acctransformer_b200 import flash_attention_packed
    q, k, v = _rows(sum(lens_q), N, D, dtype, 20), _rows(sum(lens_k), N_kv, D, dtype, 21), _rows(sum(lens_k), N_kv, D, dtype, 22)
    for causal in (True, False):
        y, lse = flash_attention_packed(q, k, v, _starts(lens_q), _starts(lens_k), causal=causal, return_lse=True)
        _check(q, k, v, lens_q, lens_k, y, lse, causal)


@pytest.mark.parametrize("B", [128, 129, 700])
def test_many_sequences(B):
    from acctransformer_b200 import flash_attention_packed
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 60, (B,), generator=g).tolist()
    lens[B // 2], lens[B - 1] = 700, 300
    T, D, dtype = sum(lens), 64, torch.float16
    q, k, v = _rows(T, 2, D, dtype, 7), _rows(T, 1, D, dtype, 8), _rows(T, 1, D, dtype, 9)
    _check(q, k, v, lens, lens, flash_attention_packed(q, k, v, _starts(lens)))


def test_every_tile_is_taken_once():
    """Sequences of all numbers of tiles, in an order that is neither ascending nor descending."""
    from acctransformer_b200 import flash_attention_packed
    g = torch.Generator().manual_seed(3)
    lens = [int(128 * i + o) for i, o in zip(torch.randperm(14, generator=g), torch.randint(-3, 4, (14,), generator=g))]
    lens = [max(0, n) for n in lens]
    prefix = torch.randint(0, 500, (14,), generator=g).tolist()
    lens_k = [n + p for n, p in zip(lens, prefix)]
    for D in (64, 128, 192):
        q, k, v = _rows(sum(lens), 3, D, torch.float16, 10), _rows(sum(lens_k), 3, D, torch.float16, 11), _rows(sum(lens_k), 3, D, torch.float16, 12)
        out = torch.full_like(q, float("nan"))
        y = flash_attention_packed(q, k, v, _starts(lens), _starts(lens_k), out=out)
        assert y.data_ptr() == out.data_ptr()
        _check(q, k, v, lens, lens_k, y)


@pytest.mark.parametrize("D", [64, 128, 160])
def test_nothing_of_other_rows_reaches_a_sequence(D):
    """The same sequences between NaNs and infinities, and between others: the same bits.  Rows of y outside are not written."""
    from acctransformer_b200 import flash_attention_packed
    dtype, N = torch.float16, 2
    lens_q, lens_k, gap = [70, 300, 1, 129], [70, 411, 30, 100], 50
    Tq, Tk = sum(lens_q), sum(lens_k)
    q, k, v = _rows(Tq, N, D, dtype, 13), _rows(Tk, N, D, dtype, 14), _rows(Tk, N, D, dtype, 15)
    want = flash_attention_packed(q, k, v, _starts(lens_q), _starts(lens_k))
    for bad in (float("nan"), float("inf"), -65504.0):
        # every second sequence is nobody's: rows of `bad`
        lq, lk = [gap], [gap]
        for a, b in zip(lens_q, lens_k):
            lq += [a, gap]
            lk += [b, gap]
        def spread(x, lens):
            out, at = [torch.full((gap,) + x.shape[1:], bad, device="cuda", dtype=dtype)], 0
            for n in lens:
                out += [x[at:at + n], out[0]]
                at += n
            return torch.cat(out)
        y = flash_attention_packed(spread(q, lens_q), spread(k, lens_k), spread(v, lens_k), _starts(lq), _starts(lk))
        at = gap
        got = []
        for n in lens_q:
            got.append(y[at:at + n])
            at += n + gap
        assert torch.equal(torch.cat(got), want)
    # one sequence in the middle of larger buffers
    cu_q, cu_k = _starts(lens_q)[1:3], _starts(lens_k)[1:3]
    out = torch.full_like(q, 7.0)
    flash_attention_packed(q, k, v, cu_q, cu_k, out=out)
    lo, hi = int(cu_q[0]), int(cu_q[1])
    assert torch.equal(out[lo:hi], want[lo:hi]) and (out[:lo] == 7).all() and (out[hi:] == 7).all()


def test_views():
    from acctransformer_b200 import flash_attention_packed
    lens, N, N_kv, D, dtype = [200, 77, 300], 8, 2, 64, torch.bfloat16
    T = sum(lens)
    q, k, v = _rows(T, N, D, dtype, 16), _rows(T, N_kv, D, dtype, 17), _rows(T, N_kv, D, dtype, 18)
    want = flash_attention_packed(q, k, v, _starts(lens))
    x = torch.cat([t.reshape(T, -1) for t in (q, k, v)], 1)
    fused = [t.view(T, -1, D) for t in x.split([N * D, N_kv * D, N_kv * D], 1)]
    heads_first = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    odd = [torch.cat([t, t[..., :1]], -1)[..., :D] for t in (q, k, v)]
    for form in (fused, heads_first, odd):
        assert torch.equal(flash_attention_packed(*form, _starts(lens)), want)
    one = k[:, :1].expand(-1, N_kv, -1)
    assert torch.equal(flash_attention_packed(q, one, one, _starts(lens)), flash_attention_packed(q, one.contiguous(), one.contiguous(), _starts(lens)))
    assert torch.equal(flash_attention_packed(q, k, v, _starts(lens).long()), want)


def test_equal_lengths_match_the_batched_op():
    """Whole tiles of one length: the same work in the same order, so the same bits."""
    from acctransformer_b200 import flash_attention_packed, flash_attention_tik
    B, S, N, D = 3, 512, 4, 128
    q, k, v = (_rows(B * S, N, D, torch.float16, s) for s in (19, 20, 21))
    y = flash_attention_packed(q, k, v, _starts([S] * B))
    b = [t.view(B, S, N, D).transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(y.view(B, S, N, D).transpose(1, 2), flash_attention_tik(*b, causal=True, scale=D ** -0.5))


def test_starts_that_make_no_sense_stay_inside_the_buffers():
    from acctransformer_b200 import _lib, flash_attention_packed
    T, N, D = 300, 2, 64
    q, k, v = (_rows(T, N, D, torch.float16, s) for s in (22, 23, 24))
    guard = torch.full((3 * T, N, D), 5.0, device="cuda", dtype=torch.float16)
    for cu in ([0, -5, 9999], [200, 100, 300], [2 ** 31 - 1, -2 ** 31, 7], [0, 0, 0]):
        flash_attention_packed(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), out=guard[T:2 * T])
    torch.cuda.synchronize()
    _lib.device_status()
    assert (guard[:T] == 5).all() and (guard[2 * T:] == 5).all()


def test_another_stream_and_a_graph():
    from acctransformer_b200 import flash_attention_packed
    lens, N, D = [300, 200], 2, 128
    q, k, v = (_rows(500, N, D, torch.float16, s) for s in (25, 26, 27))
    cu = _starts(lens)
    want = flash_attention_packed(q, k, v, cu)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        flash_attention_packed(q, k, v, cu, out=out)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    cu.copy_(_starts([100, 400]))                           # the lengths are read when it runs
    graph.replay()
    _check(q, k, v, [100, 400], [100, 400], out)


def test_behind_a_prefix_from_the_cache():
    """A chunk of a prompt whose beginning comes back from the 4-bit cache."""
    from acctransformer_b200 import Kv4Cache, flash_attention_packed
    B, N, N_kv, D, dtype = 2, 4, 2, 64, torch.float16
    prefix, chunk = [50, 17], [30, 200]
    cache = Kv4Cache(B, N_kv, 300, D, dtype=dtype)
    k0, v0 = _rows(sum(prefix), N_kv, D, dtype, 28), _rows(sum(prefix), N_kv, D, dtype, 29)
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    cache.append(k0, v0, zero, _starts(prefix))
    back = cache.read(zero, _starts(prefix), total=sum(prefix))
    q, k1, v1 = _rows(sum(chunk), N, D, dtype, 30), _rows(sum(chunk), N_kv, D, dtype, 31), _rows(sum(chunk), N_kv, D, dtype, 32)
    parts = [[torch.cat([x[a:a + p], y[b:b + c]]) for a, p, b, c in ((0, 50, 0, 30), (50, 17, 30, 200))] for x, y in zip(back, (k1, v1))]
    k, v = (torch.cat(x) for x in parts)
    lens_k = [80, 217]
    _check(q, k, v, chunk, lens_k, flash_attention_packed(q, k, v, _starts(chunk), _starts(lens_k)))


def test_refusals():
    from acctransformer_b200 import _lib, flash_attention_packed
    q = torch.zeros(10, 4, 64, device="cuda", dtype=torch.float16)
    k = q[:, :2].contiguous()
    cu = _starts([4, 6])
    bad = [
        lambda: flash_attention_packed(q, k, k[:5], cu), lambda: flash_attention_packed(q, k[:5], k[:5], cu),
        lambda: flash_attention_packed(q, q[:, :3], q[:, :3], cu), lambda: flash_attention_packed(q[0], k, k, cu),
        lambda: flash_attention_packed(q, k.bfloat16(), k, cu), lambda: flash_attention_packed(q.float(), k.float(), k.float(), cu),
        lambda: flash_attention_packed(q.cpu(), k, k, cu), lambda: flash_attention_packed(q, k, k, cu.cpu()),
        lambda: flash_attention_packed(q, k, k, cu.float()), lambda: flash_attention_packed(q, k, k, cu[:1]),
        lambda: flash_attention_packed(q, k, k, cu, cu[:2]), lambda: flash_attention_packed(q, k, k, cu, scale=-1.0),
        lambda: flash_attention_packed(q, k, k, cu, out=q[:5]), lambda: flash_attention_packed(q, k, k, cu, out=torch.zeros(10, 4, 64, device="cuda")),
        lambda: flash_attention_packed(q[..., :60].contiguous(), k[..., :60].contiguous(), k[..., :60].contiguous(), cu),
        lambda: flash_attention_packed(*(torch.zeros(10, 1, 264, device="cuda", dtype=torch.float16) for _ in range(3)), cu),
        lambda: flash_attention_packed(q.clone().requires_grad_(), k, k, cu),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, _lib.AcctError)):
            call()
            pytest.fail(f"call {i} was not refused")
    with torch.no_grad():
        flash_attention_packed(q.clone().requires_grad_(), k, k, cu)
    empty = flash_attention_packed(q[:0], k[:0], k[:0], _starts([0, 0]))
    assert empty.shape == (0, 4, 64)
