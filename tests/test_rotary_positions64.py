"""Positions of 64 bits: what does not fit in 32 is a position like any other."""
import ctypes as C

import pytest
import torch

from tests.test_rotary_far import _check


@pytest.mark.gpu
@pytest.mark.parametrize("around", [2 ** 31 - 100, 2 ** 32 - 100, 1_700_000_000_000, -2 ** 40, 2 ** 44])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_far_positions(around, dtype):
    _check(torch.arange(5000, device="cuda") + around, [1.0, 100.0, 0.0123, 10000.0 ** (-5 / 64)], dtype)


@pytest.mark.gpu
def test_types_of_the_same_positions():
    from acctransformer_b200 import Rotary
    x = torch.randn(200, 2, 64, device="cuda").bfloat16()
    rotary = Rotary(64, (16, 16))
    pos = torch.randint(0, 100, (2, 200), device="cuda")
    want = rotary(x, None, pos)[0]
    for t in (torch.int32, torch.int16, torch.int8, torch.uint8, torch.uint32):
        assert torch.equal(rotary(x, None, pos.to(t))[0], want)
    assert torch.equal(rotary(x, None, pos.t().contiguous().t())[0], want)
    high = torch.tensor([3_000_000_000], device="cuda")
    assert torch.equal(rotary(x, None, high.to(torch.uint32).expand(2, 200))[0], rotary(x, None, high.expand(2, 200))[0])


@pytest.mark.gpu
def test_gradients_and_positions_that_move_on():
    from acctransformer_b200 import Rotary
    rotary = Rotary(64, (16, 16))
    x, d = (torch.randn(3, 2, 50, 64, device="cuda").half() for _ in range(2))
    pos = torch.randint(2 ** 33, 2 ** 34, (2, 3, 50), device="cuda")
    leaf = x.clone().requires_grad_()
    y = rotary(leaf, None, pos)[0]
    (back,) = torch.autograd.grad(rotary(leaf, None, pos)[0], leaf, d)
    pos.add_(1)
    assert torch.equal(torch.autograd.grad(y, leaf, d)[0], back)
    kept = x.clone()
    rotary.apply_(kept, None, pos)
    assert torch.equal(kept, rotary(x, None, pos)[0])


def test_abi_refuses():
    from acctransformer_b200 import _lib, build
    build.build()
    lib, r = _lib.load(), _lib.RotaryArgs()
    assert lib.acct_rotary_wide(None, 4096, None) == 1
    r.dtype, r.B, r.S, r.D, r.N, r.rotated = _lib.ACCT_F16, 1, 8, 64, 2, 64
    r.q = r.q_out = r.turns = r.axis = r.positions = 4096
    assert lib.acct_rotary_wide(C.byref(r), None, None) == 1      # (those of 32 bits do not count)
    r.positions, r.D = None, 20
    assert lib.acct_rotary_wide(C.byref(r), 4096, None) == 4
