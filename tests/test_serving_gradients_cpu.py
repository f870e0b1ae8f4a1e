"""The serving operators have no gradient and say so: nothing that needs one, or carries a tangent, is taken and forgotten.  Decided
before anything looks at the device, so these run on the CPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from acctransformer_b200 import _lib, build as _build
from acctransformer_b200.infer.kv4_cache import Kv4Cache


@pytest.fixture(scope="module", autouse=True)
def _built():
    _build.build()


def _cache(slots=32):
    """A cache as its object keeps it, without the device memory that making one asks for."""
    c = Kv4Cache.__new__(Kv4Cache)
    c.B, c.N_kv, c.S_max, c.D, c.dtype, c.page_size, c.block_table = 2, 2, slots, 64, torch.float16, 0, None
    c.records = torch.zeros(2, 2, slots // 16, 1280, dtype=torch.uint8)
    c._args = (c.records, None, _lib.ACCT_F16, 2, 2, slots, 64, 0)
    return c


def _half(*shape):
    return torch.zeros(*shape, dtype=torch.float16)


class _Workspace:
    buf = torch.zeros(1 << 20, dtype=torch.uint8)


INTS = torch.zeros(2, dtype=torch.int32)


def _packed(i, x):
    from acctransformer_b200 import flash_attention_packed
    rows = [_half(4, 4, 64), _half(4, 2, 64), _half(4, 2, 64)]
    rows[i] = x(rows[i])
    flash_attention_packed(*rows, torch.tensor([0, 4], dtype=torch.int32))


CALLS = {f"packed {name}": lambda x, i=i: _packed(i, x) for i, name in enumerate("qkv")}
CALLS["append k"] = lambda x: _cache().append(x(_half(2, 2, 64)), _half(2, 2, 64), INTS)
CALLS["append v"] = lambda x: _cache().append(_half(2, 2, 64), x(_half(2, 2, 64)), INTS)
CALLS["decode q"] = lambda x: _cache().decode(x(_half(2, 4, 1, 64)), workspace=_Workspace)
CALLS["decode weights"] = lambda x: _cache().decode(_half(2, 4, 1, 64), weights=x(torch.zeros(2, 2, 32)), workspace=_Workspace)
CALLS["evict weights"] = lambda x: _cache().evict(x(torch.zeros(2, 2, 32)), INTS, 8, 2, _cache(16))


@pytest.mark.parametrize("call", CALLS.values(), ids=CALLS)
def test_what_needs_a_gradient_is_refused(call):
    with pytest.raises(ValueError, match="has no gradient"):
        call(lambda t: t.requires_grad_())
    with pytest.raises(ValueError, match="CUDA"):             # (as far as a call gets here)
        call(lambda t: t)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        call(lambda t: t.requires_grad_())
    with pytest.raises(ValueError, match="CUDA"):
        call(lambda t: t.requires_grad_().detach())


@pytest.mark.parametrize("call", CALLS.values(), ids=CALLS)
def test_what_carries_a_tangent_is_refused(call):
    with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
        call(lambda t: fwd.make_dual(t, torch.ones_like(t)))
