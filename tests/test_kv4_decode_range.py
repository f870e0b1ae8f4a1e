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
