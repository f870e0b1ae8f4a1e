"""The cache in 4 bits: rows in and out against the definition, decoding and eviction against plain implementations in 64 bits.

Tolerances are derived, not fitted.  u = 2^-11 (float16) or 2^-8 (bfloat16) is the relative error of one rounding to 16 bits.
Decoding rounds P (relative to each term), V (the same) and the result, so |y - exact| <= 3 u sum_j p_j |v_j|; the scores are
fp32 sums of products whose absolute values add up to A, so a probability is off by a factor of at most exp(2 e) with
e = 2^-20 A plus a few units of 2^-22 for the exponential and the sum."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cache(B, N_kv, S, D, dtype, page=None, seed=0):
    """A cache whose memory holds NaNs wherever a step or a minimum may lie, paged in a random order with pages to spare."""
    from acctransformer_b200 import Kv4Cache
    if page is None:
        c = Kv4Cache(B, N_kv, S, D, dtype=dtype)
    else:
        per = -(-S // page)
        order = torch.randperm(B * per + 3, generator=torch.Generator().manual_seed(seed))[:B * per]
        c = Kv4Cache(B, N_kv, S, D, dtype=dtype, page_size=page, block_table=order.int().view(B, per).cuda(), num_pages=B * per + 3)
    c.records.fill_(0xff)
    return c


def _rows(T, N_kv, D, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shift = torch.randn(N_kv, D, device="cuda", generator=g)
    return [(torch.randn(T, N_kv, D, device="cuda", generator=g) + s * shift).to(dtype) for s in (1, 0)]


def _stood_for(x):
    """The definition, in numpy on the CPU: fp32 where it says fp32, the 16-bit roundings as they are stated."""
    bf = x.dtype == torch.bfloat16
    a = x.float().cpu().numpy()
    out = np.empty_like(a)
    for at in range(0, a.shape[-1], 32):
        y = a[..., at:at + 32]
        with np.errstate(all="ignore"):
            lo, hi = y.min(-1, keepdims=True), y.max(-1, keepdims=True)      # (numpy's keep a NaN)
            want = ((hi - lo) / np.float32(15)).astype(np.float32)
            if bf:
                s = (want.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)
            else:
                h = want.astype(np.float16)
                s = np.where(h.astype(np.float32) > want, np.nextafter(h, np.float16(0)), h).astype(np.float32)
            s = np.where(np.isfinite(hi - lo), s, np.float32(np.nan))
            inv = np.where(s > 0, np.minimum(np.float32(1) / s, np.finfo(np.float32).max), np.float32(0)).astype(np.float32)
            code = np.rint(np.minimum((y - lo) * inv, np.float32(15)))
            out[..., at:at + 32] = (code.astype(np.float64) * s + lo).astype(np.float32)      # (one rounding to fp32, see below)
    return torch.from_numpy(out).to(x.dtype)


def _stood_for_exactly(x):
    """The same before the last rounding to 16 bits: what the codes, steps and minima of x say, in float64."""
    a, u = x.float(), []
    for at in range(0, a.shape[-1], 32):
        y = a[..., at:at + 32]
        lo, hi = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
        want = (hi - lo) / 15
        if x.dtype == torch.bfloat16:
            s = (want.view(torch.int32) & -65536).view(torch.float32)
        else:
            h = want.half()
            s = torch.where(h.float() > want, torch.nextafter(h.cpu(), torch.zeros((), dtype=torch.half)).to(h.device), h).float()
        code = torch.round(torch.clamp((y - lo) * torch.where(s > 0, 1 / s, 0.0), max=15.0))
        u.append(code.double() * s.double() + lo.double())
    return torch.cat(u, -1)


# ---------------------------------------------------------------------------------------------------------------------
# rows in and out
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [None, 16, 64])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 80, 96, 120, 128])
def test_rows_come_back_as_the_definition_says(D, page, dtype):
    # ragged, from one token (and none) to several records, starting inside records
    lens, start = [1, 0, 37, 16, 5, 130], [0, 3, 21, 16, 14, 7]
    B, N_kv, S = len(lens), 3, 144
    cache = _cache(B, N_kv, S, D, dtype, page)
    T = sum(lens)
    k, v = _rows(T, N_kv, D, dtype, D)
    cu = _ints(np.concatenate([[0], np.cumsum(lens)]))
    cache.append(k, v, _ints(start), cu)
    k2, v2 = cache.read(_ints(start), cu, total=T)
    # code * step + minimum is exact in 64 bits up to its last rounding; fp32 and then 16 bits is what both sides do
    assert torch.equal(k2.cpu(), _stood_for(k)) and torch.equal(v2.cpu(), _stood_for(v))


@pytest.mark.parametrize("dtype", DTYPES)
def test_special_groups(dtype):
    big = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).smallest_normal
    x = torch.zeros(10, 1, 64, device="cuda", dtype=dtype)
    x[1] = 3.25                                             # constant
    x[2, 0, 5] = float("nan")
    x[3, 0, 40] = float("inf")
    x[4, 0, 0] = -float("inf")
    x[5, 0, ::2] = -0.0
    x[6, 0, :32] = torch.linspace(-1, 1, 32).to(dtype)
    x[6, 0, 7] = big if dtype == torch.float16 else 1e30   # the largest value has to come back finite
    x[7] = (torch.arange(64) * tiny / 8).to(dtype).cuda()   # at and below the normal numbers
    x[8] = tiny / 4
    x[9, 0, 3] = tiny / 4
    cache = _cache(1, 1, 32, 64, dtype)
    cache.append(x, x.flip(0), _ints([2]), _ints([0, 10]))
    k, v = cache.read(_ints([2]), _ints([0, 10]), total=10)
    for got, given in ((k, x), (v, x.flip(0))):
        torch.testing.assert_close(got.cpu(), _stood_for(given), rtol=0, atol=0, equal_nan=True)
    assert k[2, 0, :32].isnan().all() and k[2, 0, 32:].isfinite().all()
    assert k[3, 0, 32:].isnan().all() and k[3, 0, :32].isfinite().all()
    assert k[6].isfinite().all() and k[1].eq(3.25).all()


@pytest.mark.parametrize("page", [None, 32])
def test_a_row_leaves_its_neighbours_alone(page):
    B, N_kv, S, D, dtype = 2, 2, 64, 96, torch.float16
    cache = _cache(B, N_kv, S, D, dtype, page)
    k, v = _rows(B * S, N_kv, D, dtype, 1)
    all_of, zero = _ints([0, S, 2 * S]), _ints([0, 0])
    cache.append(k, v, zero, all_of)
    want = [_stood_for(k).view(B, S, N_kv, D), _stood_for(v).view(B, S, N_kv, D)]
    for i, slot in enumerate([0, 63, 17, 30, 31, 16, 15, 46]):
        k1, v1 = _rows(B, N_kv, D, dtype, 10 + i)
        at = [slot, 63 - slot]
        cache.append(k1, v1, _ints(at))                     # one token per sequence
        for w, x in zip(want, (k1, v1)):
            for b in range(B):
                w[b, at[b]] = _stood_for(x)[b]
        one = cache.read(_ints(at))
        assert torch.equal(one[0].cpu(), _stood_for(k1)) and torch.equal(one[1].cpu(), _stood_for(v1))
    got = cache.read(zero, all_of, total=B * S)
    for g, w in zip(got, want):
        assert torch.equal(g.cpu().view(B, S, N_kv, D), w)


def test_rows_outside_the_slots_are_dropped():
    B, N_kv, S, D, dtype = 2, 1, 50, 64, torch.bfloat16
    cache = _cache(B, N_kv, S, D, dtype)
    before = cache.records.clone()
    k, v = _rows(40, N_kv, D, dtype, 2)
    cu = _ints([0, 20, 40])
    cache.append(k, v, _ints([45, -10]), cu)                # slots 45..49 and 0..9
    got, _ = cache.read(_ints([45, -10]), cu, total=40)
    assert torch.equal(got[:5].cpu(), _stood_for(k)[:5]) and torch.equal(got[30:].cpu(), _stood_for(k)[30:])
    # nothing else of the memory has changed: records 0..1 of sequence 0, 1..3 of sequence 1
    assert torch.equal(cache.records[0, 0, :2], before[0, 0, :2]) and torch.equal(cache.records[1, 0, 1:], before[1, 0, 1:])
    cache.append(k, v, _ints([50, 2 ** 31 - 1]), cu)
    cache.append(k[:0], v[:0], _ints([0, 0]), _ints([0, 0, 0]))
    cache.append(k, v, _ints([50, 60]), _ints([0, -7, 9999]))      # (starts that make no sense stay inside the rows)
    again, _ = cache.read(_ints([45, -10]), cu, total=40)
    assert torch.equal(again[:5], got[:5]) and torch.equal(again[30:], got[30:])


def test_rows_from_views():
    """k and v as parts of one projection's output, as a transposed view, and where a copy is needed."""
    B, N_kv, S, D, dtype = 3, 4, 40, 64, torch.float16
    cu, zero = _ints([0, 40, 80, 120]), _ints([0, 0, 0])
    k, v = _rows(B * S, N_kv, D, dtype, 3)
    fused = torch.cat([k, v], 1).reshape(B * S, 2 * N_kv * D)
    forms = {
        "fused": [x.view(B * S, N_kv, D) for x in fused.split(N_kv * D, 1)],
        "transposed": [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v)],
        "odd": [torch.cat([x, x[..., :1]], -1)[..., :D] for x in (k, v)],
        "expanded": [k[:, :1].expand(-1, N_kv, -1), v[:, :1].expand(-1, N_kv, -1)],
    }
    for name, (a, b) in forms.items():
        cache = _cache(B, N_kv, S, D, dtype)
        cache.append(a, b, zero, cu)
        got = cache.read(zero, cu, total=B * S)
        assert torch.equal(got[0].cpu(), _stood_for(a)) and torch.equal(got[1].cpu(), _stood_for(b)), name


# ---------------------------------------------------------------------------------------------------------------------
# decoding
# ---------------------------------------------------------------------------------------------------------------------
def _filled(lens, N_kv, S, D, dtype, page=None, seed=0):
    """A cache with lens[b] rows per sequence, and their values as float64 [B, N_kv, S, D]."""
    B, T = len(lens), sum(lens)
    cache = _cache(B, N_kv, S, D, dtype, page, seed)
    k, v = _rows(T, N_kv, D, dtype, seed)
    zero, cu = _ints([0] * B), _ints(np.concatenate([[0], np.cumsum(lens)]))
    cache.append(k, v, zero, cu)
    values = []
    for x in cache.read(zero, cu, total=T):
        full = torch.zeros(B, N_kv, S, D, dtype=torch.float64, device="cuda")
        for b, n in enumerate(lens):
            full[b, :, :n] = x[sum(lens[:b]):sum(lens[:b]) + n].double().transpose(0, 1)
        values.append(full)
    return cache, values


def _check_decode(cache, values, lens, q, y, scale, before=None, weights=None):
    k, v = values
    B, N, _, D = q.shape
    N_kv, dtype = k.shape[1], q.dtype
    u = UNIT[dtype]
    qd = q.double().view(B, N_kv, N // N_kv, D)
    y = y.double().view(B, N_kv, N // N_kv, D)
    for b, n in enumerate(lens):
        if n == 0:
            assert (y[b] == 0).all()
            assert weights is None or torch.equal(weights[b], before[b])
            continue
        kk, vv = k[b, :, :n], v[b, :, :n]
        x = scale * torch.einsum("hgd,hsd->hgs", qd[b], kk)
        A = float((scale * torch.einsum("hgd,hsd->hgs", qd[b].abs(), kk.abs())).max())
        p = torch.softmax(x, -1)
        e = 2.0 ** -20 * A + 2.0 ** -18
        k_read = 2 * u * A      # the values to compare with came back rounded to 16 bits: a relative u of every product
        want, size = p @ vv, p @ vv.abs()
        bound = size * (4 * u + math.expm1(2 * (e + k_read))) + 1e-6
        assert ((y[b] - want).abs() <= bound).all(), float(((y[b] - want).abs() / bound).max())
        if weights is not None:
            got = (weights[b, :, :n].double() - before[b, :, :n].double())
            assert ((got - p.sum(1)).abs() <= p.sum(1) * math.expm1(2 * (e + k_read)) + before[b, :, :n].abs() * 2.0 ** -23 + 1e-9).all()
            assert torch.equal(weights[b, :, n:], before[b, :, n:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [None, 32])
@pytest.mark.parametrize("D, group", [(128, 1), (128, 4), (128, 8), (128, 9), (128, 16), (64, 1), (64, 7), (96, 3), (80, 12), (40, 5), (32, 2), (8, 1)])
def test_decode_against_64_bits(D, group, page, dtype):
    lens = [0, 1, 15, 16, 17, 64, 129, 700]
    N_kv, S = 2, 704
    cache, values = _filled(lens, N_kv, S, D, dtype, page, seed=D + group)
    g = torch.Generator(device="cuda").manual_seed(group)
    q = torch.randn(len(lens), N_kv * group, 1, D, device="cuda", generator=g).to(dtype)
    weights = torch.rand(len(lens), N_kv, cache.S_max, device="cuda", generator=g)
    before = weights.clone()
    y = cache.decode(q, _ints(lens), weights=weights)
    assert y.shape == q.shape and y.dtype == dtype
    _check_decode(cache, values, lens, q, y, D ** -0.5, before, weights)
    plain = cache.decode(q, _ints(lens))
    assert torch.equal(plain, y)


@pytest.mark.parametrize("splits", [0, 1, 3, 64])
def test_decode_in_parts(splits):
    from acctransformer_b200 import Kv4Workspace
    lens, N_kv, D, dtype = [2000, 65, 1], 2, 128, torch.float16
    cache, values = _filled(lens, N_kv, 2000, D, dtype, seed=5)
    q = torch.randn(3, 8, 1, D, device="cuda").to(dtype)
    ws = Kv4Workspace(3, 8, N_kv, 2000, D, "cuda", weights=True, num_splits=splits)
    ws.buf.fill_(0xff)
    weights = torch.zeros(3, N_kv, 2000, device="cuda")
    out = torch.empty_like(q)
    y = cache.decode(q, _ints(lens), scale=0.2, weights=weights, num_splits=splits, workspace=ws, out=out)
    assert y.data_ptr() == out.data_ptr()
    _check_decode(cache, values, lens, q, y, 0.2, torch.zeros_like(weights), weights)
    total = weights.sum(-1)
    torch.testing.assert_close(total, torch.full_like(total, 4.0), rtol=1e-5, atol=0)      # four query heads' probabilities


def test_decode_is_reproducible_and_runs_on_the_callers_stream():
    lens, N_kv, D, dtype = [513, 4096, 77], 4, 128, torch.bfloat16
    cache, _ = _filled(lens, N_kv, 4096, D, dtype, 64, seed=6)
    q = torch.randn(3, 16, 1, D, device="cuda").to(dtype)
    runs = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            w = torch.zeros(3, N_kv, cache.S_max, device="cuda")
            runs.append((cache.decode(q, _ints(lens), weights=w), w))
        torch.cuda.synchronize()
    for y, w in runs[1:]:
        assert torch.equal(y, runs[0][0]) and torch.equal(w, runs[0][1])


def test_what_lies_past_the_length_does_not_matter():
    """Rows of NaNs and infinities behind the length, inside its last record."""
    lens, N_kv, S, D, dtype = [5, 20], 1, 32, 64, torch.float16
    cache, values = _filled([32, 32], N_kv, S, D, dtype, seed=7)
    bad = torch.full((44, N_kv, D), float("nan"), device="cuda", dtype=dtype)
    bad[::2] = float("inf")
    cache.append(bad[:39], bad[:39], _ints(lens), _ints([0, 27, 39]))
    q = torch.randn(2, 3, 1, D, device="cuda").to(dtype)
    w = torch.zeros(2, N_kv, S, device="cuda")
    y = cache.decode(q, _ints(lens), weights=w)
    _check_decode(cache, values, lens, q, y, D ** -0.5, torch.zeros_like(w), w)
    # a NaN inside the length does reach the result
    y = cache.decode(q, _ints([6, 20]))
    assert y[0].isnan().all() and y[1].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 8])
def test_probabilities_keep_more_than_16_bits(group, dtype):
    """V in 0..15 with both in every group of 32, step 1 and minimum 0: its values are exact.  P is a sum of two 16-bit numbers up to a
    group of 8 (a relative u^2; in float16 a half unit of its smallest number, 2^-25, for each), so little but the last
    rounding is left."""
    lens, N_kv, S, D, u = [5, 40, 300], 2, 300, 128, UNIT[dtype]
    T = sum(lens)
    cache = _cache(3, N_kv, S, D, dtype, seed=21)
    g = torch.Generator(device="cuda").manual_seed(group)
    k, v = _rows(T, N_kv, D, dtype, 21)[0], torch.randint(0, 16, (T, N_kv, D), device="cuda", generator=g).to(dtype)
    v[..., 0::32], v[..., 1::32] = 0, 15
    zero, cu = _ints([0] * 3), _ints([0, 5, 45, 345])
    cache.append(k, v, zero, cu)
    _, v_read = cache.read(zero, cu, total=T)
    assert torch.equal(v_read, v)
    q = (0.5 * torch.randn(3, N_kv * group, 1, D, device="cuda", generator=g)).to(dtype)
    w = torch.zeros(3, N_kv, S, device="cuda")
    y = cache.decode(q, _ints(lens), weights=w)
    for b, n in enumerate(lens):
        at = sum(lens[:b])
        for h in range(N_kv):
            qq, kk, vv = (x.double() for x in (q[b, h * group:(h + 1) * group, 0], _stood_for_exactly(k[at:at + n, h]).cuda(), v[at:at + n, h]))
            p = torch.softmax(qq @ kk.T * D ** -0.5, -1)
            e = 2.0 ** -20 * float((qq.abs() @ kk.abs().T * D ** -0.5).max()) + 2.0 ** -18
            want = p @ vv
            room = want * (u * u + math.expm1(2 * e)) + n * 15 * 2.0 ** -25
            got = y[b, h * group:(h + 1) * group, 0].double()
            assert ((got - want).abs() <= u * (want + room) + room).all(), float(((got - want).abs() / (u * want)).max())


def test_steps_in_a_graph():
    """Writing, decoding and eviction captured once and replayed on new contents: as the calls themselves give it."""
    B, N_kv, D, S, dtype = 3, 2, 64, 200, torch.float16
    lens = [200, 90, 1]
    zero, cu = _ints([0] * B), _ints([0, 200, 290, 291])
    k, v = _rows(291, N_kv, D, dtype, 31)
    q = torch.randn(B, 8, 1, D, device="cuda").to(dtype)
    w = torch.zeros(B, N_kv, S, device="cuda")
    seq = _ints(lens)
    cache, spare = _cache(B, N_kv, S, D, dtype, seed=1), _cache(B, N_kv, 64, D, dtype, seed=2)

    def steps():
        w.zero_()
        cache.append(k, v, zero, cu)
        y = cache.decode(q, seq, weights=w)
        return (y, w.clone(), *cache.evict(w, seq, 64, 5, spare), *spare.read(zero, cu[:4].clamp(max=64), total=64))

    steps()      # (what a first call sets up)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = steps()
    for seed in (32, 33):
        for x, y in zip((k, v), _rows(291, N_kv, D, dtype, seed)):
            x.copy_(y)
        q.copy_(torch.randn(q.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
        want = [x.clone() for x in steps()]
        for x in out:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for i, (x, y) in enumerate(zip(out, want)):
            assert torch.equal(x, y), i


def test_the_example(tmp_path):
    """The example's loop, small enough to fill and evict twice; decoding there agrees with attention over the same rows to what 16-bit
    values of K and V, P and the result differ by: 4 roundings of 2^-9 rms, and as much again for the scores."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "serve_kv4.py")
    spec = importlib.util.spec_from_file_location("serve_kv4", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    r = module.serve(layers=2, batch=3, slots=96, tokens=120, hidden=128)
    assert r["evictions"] >= 2 and max(r["lens"]) <= 96 and r["difference"] < 8 * 2.0 ** -9 and r["out"].isfinite().all()
    assert r["cache_bytes"] < 0.33 * r["bytes_in_16_bits"]


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_and_small_queries(dtype):
    """Scores far apart (one key takes everything) and all alike."""
    lens, N_kv, D = [200, 33], 1, 128
    cache, values = _filled(lens, N_kv, 200, D, dtype, seed=8)
    for size in (1e-4, 30.0):
        q = (size * torch.randn(2, 2, 1, D, device="cuda")).to(dtype)
        y = cache.decode(q, _ints(lens))
        _check_decode(cache, values, lens, q, y, D ** -0.5)


def test_offsets_past_32_bits():
    """A cache of over 4 GB, of which the last sequence is used; and a pool of pages of which the last are."""
    from acctransformer_b200 import Kv4Cache
    B, N_kv, S, D, dtype = 40, 64, 16384, 64, torch.float16
    cache = Kv4Cache(B, N_kv, S, D, dtype=dtype)
    assert cache.nbytes > 2 ** 31
    n = 40
    k, v = _rows(n, N_kv, D, dtype, 9)
    cu = _ints([0] * B + [n])
    start = _ints([0] * (B - 1) + [S - n])
    cache.append(k, v, start, cu)
    got = cache.read(start, cu, total=n)
    assert torch.equal(got[0].cpu(), _stood_for(k)) and torch.equal(got[1].cpu(), _stood_for(v))
    del cache
    pages = 80000
    table = _ints([[pages - 1, pages - 2]])
    cache = Kv4Cache(1, N_kv, 32, D, dtype=dtype, page_size=16, block_table=table, num_pages=pages)
    assert cache.nbytes > 2 ** 32
    cache.append(k[:32], v[:32], _ints([0]), _ints([0, 32]))
    got = cache.read(_ints([0]), _ints([0, 32]), total=32)
    assert torch.equal(got[0].cpu(), _stood_for(k[:32]))
    values = [x.double().transpose(0, 1)[None] for x in got]
    q = torch.randn(1, N_kv, 1, D, device="cuda").to(dtype)
    _check_decode(cache, values, [31], q, cache.decode(q, _ints([31])), D ** -0.5)


def test_pages_outside_the_pool_touch_no_other_memory():
    from acctransformer_b200 import Kv4Cache
    table = _ints([[0, -5, 2 ** 31 - 1, 1]])
    cache = Kv4Cache(1, 1, 64, 64, dtype=torch.float16, page_size=16, block_table=table, num_pages=2)
    k, v = _rows(64, 1, 64, torch.float16, 10)
    cache.append(k[:16], v[:16], _ints([0]), _ints([0, 16]))
    got, _ = cache.read(_ints([0]), _ints([0, 32]), total=32)
    assert torch.equal(got[:16], got[16:])                  # page -5 stands for page 0
    cache.append(k[:16], v[:16], _ints([48]), _ints([0, 16]))
    assert cache.decode(torch.randn(1, 1, 1, 64, device="cuda").half(), _ints([64])).isfinite().all()


# ---------------------------------------------------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------------------------------------------------
def _evicted(w, lens, keep, recent):
    """[B, N_kv, keep] kept slots, by sorting on the CPU."""
    w = w.cpu().double().numpy()
    out = np.full(w.shape[:2] + (keep,), -1, dtype=np.int64)
    for b, n in enumerate(lens):
        for h in range(w.shape[1]):
            old = max(0, n - recent)
            x = np.where(np.isnan(w[b, h, :old]), np.inf, w[b, h, :old])
            nan = np.isnan(w[b, h, :old])
            best = np.lexsort((np.arange(old), -x, ~nan))[:max(0, min(n, keep) - (n - old))]
            slots = np.concatenate([np.sort(best), np.arange(old, n)])
            out[b, h, :len(slots)] = slots
    return torch.from_numpy(out)


def _check_evict(cache, spare, w, lens, keep, recent):
    B, N_kv = w.shape[:2]
    kept, w2, lens2 = cache.evict(w, _ints(lens), keep, recent, spare)
    want = _evicted(w, lens, keep, recent)
    assert kept.dtype == torch.int32 and torch.equal(kept.cpu().long(), want)
    n2 = [min(n, keep) for n in lens]
    assert lens2.tolist() == n2
    assert w2.shape == (B, N_kv, spare.S_max)
    got_w = torch.where(want >= 0, w.cpu().gather(-1, want.clamp(min=0)), torch.tensor(0.0))
    torch.testing.assert_close(w2[..., :keep].cpu(), got_w, rtol=0, atol=0, equal_nan=True)
    assert (w2[..., keep:] == 0).all()
    # the rows themselves, bit for bit
    def contents(c, counts):
        k, v = c.read(_ints([0] * B), _ints(np.concatenate([[0], np.cumsum(counts)])), total=sum(counts))
        at = np.concatenate([[0], np.cumsum(counts)])
        return [[x[at[b]:at[b + 1]] for b in range(B)] for x in (k, v)]
    for old, new in zip(contents(cache, lens), contents(spare, n2)):
        for b in range(B):
            for h in range(N_kv):
                assert torch.equal(new[b][:, h], old[b][want[b, h, :n2[b]].cuda(), h])
    return kept, w2, lens2


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [None, 16])
@pytest.mark.parametrize("D", [32, 64, 80, 128])
def test_evict_against_a_sort(D, page, dtype):
    lens, N_kv, S = [0, 1, 30, 31, 200, 333], 2, 336
    cache, _ = _filled(lens, N_kv, S, D, dtype, page, seed=D)
    g = torch.Generator(device="cuda").manual_seed(D)
    w = torch.randn(len(lens), N_kv, cache.S_max, device="cuda", generator=g).exp()
    for keep, recent in ((30, 7), (1, 0), (1, 1), (17, 17), (100, 0), (333, 50)):
        spare = _cache(len(lens), N_kv, keep + 3, D, dtype, page, seed=1)
        _check_evict(cache, spare, w, lens, keep, recent)


def test_evict_ties_and_odd_weights():
    lens, N_kv, S, D, dtype = [300, 300, 257, 64], 2, 300, 64, torch.float16
    cache, _ = _filled(lens, N_kv, S, D, dtype, seed=2)
    w = torch.randint(0, 3, (4, N_kv, S), device="cuda").float()        # many of each
    w[1] = 0.0                                                          # all alike
    w[2, 0, 5::7] = float("nan")
    w[2, 1, ::3] = float("inf")
    w[2, 1, 1::3] = -float("inf")
    w[3, 0, ::2] = -0.0
    w[3, 1] = -w[3, 1] - 1e-40
    for keep, recent in ((64, 16), (100, 99), (250, 0), (37, 1)):
        _check_evict(cache, _cache(4, N_kv, keep, D, dtype), w, lens, keep, recent)


@pytest.mark.parametrize("S", [2048, 2049, 8192, 9000, 16384, 16385, 50000, 60001])
def test_evict_long(S):
    N_kv, D, dtype = 2, 32, torch.float16
    lens = [S, S - 1]
    cache, _ = _filled(lens, N_kv, S, D, dtype, seed=3)
    g = torch.Generator(device="cuda").manual_seed(S)
    w = torch.randn(2, N_kv, S, device="cuda", generator=g).exp()
    w[0, 1] = (w[0, 1] * 8).round()                                     # ties
    for keep, recent in ((S // 2, 100), (33, 0), (S - 5, S // 3)):
        _check_evict(cache, _cache(2, N_kv, keep, D, dtype), w, lens, keep, recent)


def test_a_serving_loop():
    """Prompts, decoding steps that add up probabilities, eviction when the cache is full, and on: against the same in 64 bits."""
    B, N_kv, group, D, S, dtype = 2, 2, 4, 64, 96, torch.float16
    caches = [_cache(B, N_kv, S, D, dtype, seed=4) for _ in range(2)]
    g = torch.Generator(device="cuda").manual_seed(11)
    lens = [60, 41]
    k, v = _rows(sum(lens), N_kv, D, dtype, 12)
    seq = _ints([0, 0])
    caches[0].append(k, v, seq, _ints([0, lens[0], sum(lens)]))
    seq += _ints(lens)
    w = torch.zeros(B, N_kv, S, device="cuda")
    vals = [[_stood_for(x).double()[:60], _stood_for(x).double()[60:]] for x in (k, v)]      # [k, v][b]: [n, N_kv, D]
    vals = [[[x[b][:, h] for h in range(N_kv)] for b in range(B)] for x in vals]
    w64 = [[torch.zeros(lens[b], dtype=torch.float64) for _ in range(N_kv)] for b in range(B)]
    for step in range(80):
        if max(lens) == S:
            kept, w, seq = caches[0].evict(w, seq, 48, 10, caches[1])
            caches.reverse()
            assert w.shape[-1] == S
            for b in range(B):
                for h in range(N_kv):
                    at = kept[b, h][kept[b, h] >= 0].cpu().long()
                    n = lens[b]
                    best = set(w64[b][h][:n - 10].topk(min(n, 48) - 10).indices.tolist()) if n > 48 else set(range(n - 10))
                    # (which of two that are equal up to the roundings stays is not determined)
                    cut = min((float(w64[b][h][i]) for i in best), default=0.0)
                    for i in set(at.tolist()) ^ (best | set(range(n - 10, n))):
                        assert abs(float(w64[b][h][i]) - cut) < 2e-3 * cut
                    for x in vals:
                        x[b][h] = x[b][h][at]
                    w64[b][h] = w64[b][h][at]
                lens[b] = min(lens[b], 48)
            assert seq.tolist() == lens
        k1, v1 = _rows(B, N_kv, D, dtype, 100 + step)
        caches[0].append(k1, v1, seq)
        seq = seq + 1
        lens = [n + 1 for n in lens]
        q = torch.randn(B, N_kv * group, 1, D, device="cuda", generator=g).to(dtype)
        y = caches[0].decode(q, seq, weights=w)
        for b in range(B):
            for h in range(N_kv):
                for x, new in zip(vals, (k1, v1)):
                    x[b][h] = torch.cat([x[b][h], _stood_for(new)[b, h].double()[None]])
                qq = q[b, h * group:(h + 1) * group, 0].double().cpu()
                p = torch.softmax(qq @ vals[0][b][h].T / math.sqrt(D), -1)
                want = p @ vals[1][b][h]
                assert (y[b, h * group:(h + 1) * group, 0].double().cpu() - want).abs().max() < 1e-2
                w64[b][h] = torch.cat([w64[b][h], torch.zeros(1, dtype=torch.float64)]) + p.sum(0)
                torch.testing.assert_close(w[b, h, :lens[b]].cpu().double(), w64[b][h], rtol=2e-3, atol=1e-6)


def test_refusals():
    from acctransformer_b200 import Kv4Cache, Kv4Workspace, _lib
    half = torch.float16
    cache = _cache(2, 2, 32, 64, half)
    q = torch.zeros(2, 4, 1, 64, device="cuda", dtype=half)
    k = torch.zeros(2, 2, 64, device="cuda", dtype=half)
    zero, w = _ints([0, 0]), torch.zeros(2, 2, 32, device="cuda")
    spare = _cache(2, 2, 16, 64, half)
    bad = [
        lambda: Kv4Cache(1, 1, 16, 136), lambda: Kv4Cache(1, 1, 16, 60), lambda: Kv4Cache(1, 1, 0, 64),
        lambda: Kv4Cache(1, 1, 16, 64, dtype=torch.float32), lambda: Kv4Cache(1, 1, 16, 64, device="cpu"),
        lambda: Kv4Cache(1, 1, 16, 64, page_size=16), lambda: Kv4Cache(1, 1, 16, 64, page_size=24, block_table=_ints([[0]])),
        lambda: Kv4Cache(1, 1, 17, 64, page_size=16, block_table=_ints([[0]])),
        lambda: Kv4Cache(1, 1, 16, 64, page_size=16, block_table=_ints([[0]]).long()),
        lambda: cache.append(k.bfloat16(), k.bfloat16(), zero), lambda: cache.append(k[:1], k[:1], zero),
        lambda: cache.append(k[:, :1], k[:, :1], zero), lambda: cache.append(k, k[:1], zero), lambda: cache.append(k.cpu(), k.cpu(), zero),
        lambda: cache.append(k, k, zero.cpu()), lambda: cache.append(k, k, zero[:1]), lambda: cache.append(k, k, zero, zero),
        lambda: cache.append(k, k, zero.float()),
        lambda: cache.read(zero, _ints([0, 1, 2])), lambda: cache.read(zero, total=3),
        lambda: cache.decode(q[:, :3]), lambda: cache.decode(q[:1]), lambda: cache.decode(q.bfloat16()), lambda: cache.decode(q.cpu()),
        lambda: cache.decode(q.expand(2, 4, 2, 64)), lambda: cache.decode(q, zero.cpu()), lambda: cache.decode(q, zero[:1]),
        lambda: cache.decode(q, weights=w[..., :31]), lambda: cache.decode(q, weights=w.half()), lambda: cache.decode(q, out=q[:1]),
        lambda: cache.decode(q, scale=0.0), lambda: cache.decode(q, num_splits=65),
        lambda: cache.decode(torch.zeros(2, 34, 1, 64, device="cuda", dtype=half)),
        lambda: cache.decode(q, weights=w, workspace=Kv4Workspace(2, 4, 2, 32, 64, "cuda", num_splits=1)),
        lambda: cache.evict(w, zero, 17, 0, spare), lambda: cache.evict(w, zero, 8, 9, spare), lambda: cache.evict(w, zero, 0, 0, spare),
        lambda: cache.evict(w, zero, 8, -1, spare), lambda: cache.evict(w, zero, 8, 0, cache), lambda: cache.evict(w, zero, 8, 0, w),
        lambda: cache.evict(w, zero, 8, 0, _cache(2, 1, 16, 64, half)), lambda: cache.evict(w, zero, 8, 0, _cache(2, 2, 16, 64, torch.bfloat16)),
        lambda: cache.evict(w[:1], zero, 8, 0, spare), lambda: cache.evict(w.double(), zero, 8, 0, spare),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, _lib.AcctError)):
            call()
            pytest.fail(f"call {i} was not refused")
    assert (cache.decode(q, zero) == 0).all()               # and the cache works on
