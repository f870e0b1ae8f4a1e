"""Rotary positions without rows: new tensors, like those with rows."""
import pytest
import torch

from tests.test_linear_attention import _ours

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,at", [((0, 2, 64), (2, 0)), ((3, 2, 0, 64), (2, 0)), ((0, 2, 5, 64), (2, 5)), ((0, 2, 5, 64), (2, 0, 5))])
def test_results_are_new(shape, at):
    rotary = _ours().Rotary(64, (16, 16))
    q, k = (torch.zeros(shape, device="cuda", dtype=torch.float16).requires_grad_() for _ in range(2))
    pos = torch.zeros(at, dtype=torch.int32, device="cuda")
    y = rotary(q, k, pos)
    assert all(a.shape == shape and a is not x and not a.is_leaf for a, x in zip(y, (q, k)))
    grads = torch.autograd.grad(y, (q, k), [torch.zeros_like(a) for a in y])
    assert all(g.shape == shape for g in grads)
    with torch.no_grad():
        assert rotary(q, None, pos)[0] is not q and rotary(q, None, pos)[1] is None
        assert rotary.apply_(q, k, pos)[0] is q
