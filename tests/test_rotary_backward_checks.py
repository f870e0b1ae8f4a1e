"""What the backward of rotary positions is handed by hooks on saved tensors and on gradients is checked like what the forward was given."""
import pytest
import torch

from tests.test_linear_attention import _ours, _rand

pytestmark = pytest.mark.gpu

T, N, D = 300, 2, 64


def _turned(hook=lambda t: t, axes=2):
    rotary = _ours().Rotary(D, (16,) * axes)
    x = _rand(T, N, D, dtype=torch.float16, seed=1).requires_grad_()
    pos = torch.randint(0, 500, (axes, T), device="cuda", dtype=torch.int32)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, hook):
        return x, rotary(x, None, pos)[0], pos, rotary


CHANGED = {"long": lambda t: t.long(), "host": lambda t: t.cpu(), "few": lambda t: t[..., :-1], "axes": lambda t: t[:1], "float": lambda t: t.float(),
           "flat": lambda t: t.flatten()}


@pytest.mark.parametrize("change", sorted(CHANGED))
def test_other_positions_are_refused(change):
    x, y, _, _ = _turned(CHANGED[change])
    with pytest.raises(ValueError, match="positions"):
        torch.autograd.grad(y, x, torch.ones_like(y))


def test_copies_are_taken():
    x, y, pos, rotary = _turned(lambda t: t.clone() if t.dim() != 3 else t.transpose(0, 2).contiguous().transpose(0, 2))
    d = _rand(T, N, D, dtype=torch.float16, seed=2)
    (got,) = torch.autograd.grad(y, x, d)
    assert torch.equal(got, torch.autograd.grad(rotary(x, None, pos)[0], x, d)[0])


def test_other_gradients_are_refused():
    for change in (lambda g: g[:-1], lambda g: g[..., :32], lambda g: g.float()):
        x, y, _, _ = _turned()
        y.register_hook(change)
        with pytest.raises((ValueError, RuntimeError)):
            torch.autograd.grad(y, x, torch.ones_like(y))
