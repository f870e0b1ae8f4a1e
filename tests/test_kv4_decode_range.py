"""Decoding over the 4-bit cache where queries or scores are far from the usual size: what is small keeps its bits, and what is out of
fp32's range counts for nothing, as in the definition."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _exact_rows(T, N_kv, D, dtype, seed):
    """Integers 0..15 with both ends in every group of 32: step 1 and minimum 0, so that the cache holds them as they are."""
    x = torch.randint(0, 16, (T, N_kv, D), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)
    x[..., 0::32], x[..., 1::32] = 0, 15
    return x


@pytest.mark.parametrize("D", [128, 40])
@pytest.mark.parametrize("group", [1, 4, 7, 16])
@pytest.mark.parametrize("size", [2.0 ** -24, 1e-6, 1e-5, 1e-4, 2.0 ** -10, 1.0, 2.0 ** 12])
def test_queries_of_any_size(size, group, D):
    """q of the given size with a scale that brings the scores back, in float16, whose small numbers have few bits: q is exact as it is
    given, so its size may not matter.  Heads of one group differ in size, too.  K and V are exact in the cache: K = code - 7.

    Roundings: P to 16 bits (up to 8 heads twice, the second time what the first has left) and the result, u = 2^-11 each; half a unit
    of the smallest number, 2^-25, for each of P's; scores off by e = 2^-20 A: fp32 sums of q code and 7 q, whose absolute values
    add up to A (2^-34 of the largest q that may be left out of each q is far below that), so a probability by a factor of exp(2 e)."""
    lens, N_kv, S, dtype, u = [5, 40, 300], 2, 300, torch.float16, 2.0 ** -11
    from acctransformer_b200 import Kv4Cache
    T = sum(lens)
    cache = Kv4Cache(3, N_kv, S, D, dtype=dtype)
    k, v = _exact_rows(T, N_kv, D, dtype, 1) - 7, _exact_rows(T, N_kv, D, dtype, 2)
    zero, cu = _ints([0] * 3), _ints([0, 5, 45, 345])
    cache.append(k, v, zero, cu)
    back = cache.read(zero, cu, total=T)
    assert torch.equal(back[0], k) and torch.equal(back[1], v)
    g = torch.Generator(device="cuda").manual_seed(group)
    q = torch.randn(3, N_kv * group, 1, D, device="cuda", generator=g)
    q = (size * q * 2.0 ** -(torch.arange(N_kv * group, device="cuda") % 3)[None, :, None, None]).to(dtype)
    scale = 0.1 * D ** -0.5 / size
    w = torch.zeros(3, N_kv, S, device="cuda")
    y = cache.decode(q, _ints(lens), scale=scale, weights=w)
    for b, n in enumerate(lens):
        at = sum(lens[:b])
        for h in range(N_kv):
            qq, kk, vv = (x.double() for x in (q[b, h * group:(h + 1) * group, 0], k[at:at + n, h], v[at:at + n, h]))
            p = torch.softmax(scale * qq @ kk.T, -1)
            e = 2.0 ** -20 * float((scale * qq.abs() @ (kk + 14).T).max()) + 2.0 ** -18
            want = p @ vv
            room = want * ((u if group > 8 else u * u) + math.expm1(2 * e)) + n * 15 * 2.0 ** -25
            got = y[b, h * group:(h + 1) * group, 0].double()
            assert ((got - want).abs() <= u * (want + room) + room).all(), float(((got - want).abs() / (u * want)).max())
            assert ((w[b, h, :n].double() - p.sum(0)).abs() <= p.sum(0) * (math.expm1(2 * e) + group * 2.0 ** -22) + 1e-9).all()


@pytest.mark.parametrize("page", [None, 32])
@pytest.mark.parametrize("group", [1, 4, 8, 16])
@pytest.mark.parametrize("splits", [0, 1, 5])
def test_scores_below_the_range_of_fp32(splits, group, page):
    """Keys at the lowest value of bfloat16, whose scores are -inf in fp32: weight 0, however many of them come together (whole
    warps' shares, whole parts), and everywhere but in one sequence: only the others count.  Of the last sequence no key is left."""
    from acctransformer_b200 import Kv4Cache
    dtype, N_kv, S, D = torch.bfloat16, 2, 704, 64
    lens = [700, 100, 33, 640]
    B, T = len(lens), sum(lens)
    table = {} if page is None else {"page_size": page, "block_table": torch.randperm(B * S // page).int().view(B, -1).cuda()}
    cache = Kv4Cache(B, N_kv, S, D, dtype=dtype, **table)
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(T, N_kv, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    there = [range(300, 411), [99], [0], []]                 # keys with a score in range
    at = 0
    for n, some in zip(lens, there):
        hidden = torch.ones(n, dtype=torch.bool, device="cuda")
        hidden[list(some)] = False
        k[at:at + n][hidden] = torch.finfo(dtype).min
        at += n
    zero, cu = _ints([0] * B), torch.tensor([0] + lens).cumsum(0).int().cuda()
    cache.append(k, v, zero, cu)
    k, v = cache.read(zero, cu, total=T)
    q = (1.0 + torch.rand(B, N_kv * group, 1, D, device="cuda", generator=g)).to(dtype)
    w = torch.zeros(B, N_kv, cache.S_max, device="cuda")
    y = cache.decode(q, _ints(lens), weights=w, num_splits=splits)
    at = 0
    for b, (n, some) in enumerate(zip(lens, there)):
        some = list(some)
        for h in range(N_kv):
            got, p_got = y[b, h * group:(h + 1) * group, 0].double(), w[b, h].double()
            if not some:
                assert (got == 0).all() and (p_got == 0).all()
                continue
            qq, kk, vv = (x.double() for x in (q[b, h * group:(h + 1) * group, 0], k[at:at + n, h][some], v[at:at + n, h][some]))
            x = qq @ kk.T * D ** -0.5
            p = torch.softmax(x, -1)
            # u = 2^-8: V and the result rounded (and P, above 8 heads); K came back rounded, a relative u of every product
            u, A = 2.0 ** -8, float((qq.abs() @ kk.abs().T).max()) * D ** -0.5
            change = math.expm1(2 * (2.0 ** -20 * A + 2.0 ** -18 + 2 * u * A))
            assert ((got - p @ vv).abs() <= (p @ vv.abs()) * (4 * u + change) + 1e-6).all()
            assert ((p_got[some] - p.sum(0)).abs() <= p.sum(0) * change + 1e-9).all()
            p_got[some] = 0
            assert (p_got == 0).all()
        at += n
