"""Rotary positions with several axes on the GPU against the formula in 64 bits.

Tolerances: the sine and cosine are off by at most 2^-22 (24 bits of the angle, which as a fraction of a turn is off by 2^-24 of half a
turn, and two units in the last place), each of the three fp32 operations of an output by 2^-24 of its terms, and the output is rounded
once: u |y| + 2^-21 (|x1| + |x2|)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _turned(x, pos, sections, base=10000.0, per_axis=False, adjacent=False, frequencies=None, sign=1.0):
    """x [..., D] with angles from pos [axes, ...]: (values, the sums of the absolute values that go into them) in float64."""
    pairs = sum(sections)
    if frequencies is None:
        frequencies = [base ** (-i / n) for n in sections for i in range(n)] if per_axis else [base ** (-i / pairs) for i in range(pairs)]
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    x = x.double()
    y, most = x.clone(), torch.zeros_like(x)
    for i in range(pairs):
        a, b = (2 * i, 2 * i + 1) if adjacent else (i, i + pairs)
        w = pos[axis[i]].double() * frequencies[i] * sign
        c, s = torch.cos(w), torch.sin(w)
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
        most[..., a] = most[..., b] = x[..., a].abs() + x[..., b].abs()
    return y, most


def _check(got, want, most):
    u = torch.finfo(got.dtype).eps / 2
    bound = u * want.abs() + 2.0 ** -21 * most + torch.finfo(got.dtype).tiny
    assert ((got.double() - want).abs() <= bound).all()


CASES = [
    dict(D=128, sections=(64,)), dict(D=128, sections=(16, 24, 24)), dict(D=80, sections=(16, 16), adjacent=True, per_axis=True),
    dict(D=40, sections=(7, 6, 7)), dict(D=64, sections=(5,)), dict(D=256, sections=(1, 127), adjacent=True), dict(D=8, sections=(0, 4)),
    dict(D=96, sections=(12, 10), adjacent=True, base=500000.0), dict(D=72, sections=(3, 3), adjacent=True)]


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c['D']}-{c['sections']}")
@pytest.mark.parametrize("T,N,N_kv,far", [(1, 1, 1, 100), (37, 5, 2, 1 << 20), (700, 8, 8, 2 ** 31 - 1)])
def test_packed_rows(dt, case, T, N, N_kv, far):
    from acctransformer_b200 import Rotary
    case = dict(case)
    D, sections = case.pop("D"), case.pop("sections")
    torch.manual_seed(T)
    q, k = (torch.randn(T, h, D, device="cuda").to(DTYPES[dt]) for h in (N, N_kv))
    pos = torch.randint(-far if far < 2 ** 31 - 1 else 0, far, (len(sections), T), device="cuda", dtype=torch.int32)
    rotary = Rotary(D, sections, **case)
    out = rotary(q, k, pos)
    for x, y in zip((q, k), out):
        want, most = _turned(x, pos[..., None].expand(-1, -1, x.shape[1]), sections, **case)
        # positions up to 2^31 times a frequency with 53 bits, in float64 here: 2^-20 of the angle's sine at most
        _check(y, want, most * (4 if far > 1 << 20 else 1))
    for i, only in enumerate((rotary(q, None, pos)[0], rotary(None, k, pos)[1])):
        assert torch.equal(only, out[i])
    inplace = [q.clone(), k.clone()]
    got = rotary.apply_(*inplace, pos)
    assert got[0].data_ptr() == inplace[0].data_ptr() and all(torch.equal(a, b) for a, b in zip(inplace, out))


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("shared", [False, True])
def test_batches_and_gradients(dt, shared):
    from acctransformer_b200 import Rotary
    B, N, N_kv, S, D, sections = 3, 4, 2, 65, 64, (6, 10, 4)
    torch.manual_seed(1)
    q, dq = (torch.randn(B, N, S, D, device="cuda").to(DTYPES[dt]) for _ in range(2))
    k, dk = (torch.randn(B, N_kv, S, D, device="cuda").to(DTYPES[dt]) for _ in range(2))
    pos = torch.randint(0, 5000, (3, S) if shared else (3, B, S), device="cuda", dtype=torch.int64)
    at = (pos[:, None] if shared else pos)[:, :, None].expand(-1, B, N, S)
    q.requires_grad_()
    k.requires_grad_()
    rotary = Rotary(D, sections)
    y = rotary(q, k, pos)
    for x, t in zip((q, k), y):
        _check(t.detach(), *_turned(x.detach(), at[:, :, :x.shape[1]], sections))
    for g, d in zip(torch.autograd.grad(y, (q, k), (dq, dk)), (dq, dk)):
        _check(g, *_turned(d, at[:, :, :d.shape[1]], sections, sign=-1.0))
    # one of the two alone, with an output gradient in another layout
    (g,) = torch.autograd.grad(rotary(q, None, pos)[0], q, dq.transpose(1, 2).contiguous().transpose(1, 2))
    _check(g, *_turned(dq, at[:, :, :N], sections, sign=-1.0))
