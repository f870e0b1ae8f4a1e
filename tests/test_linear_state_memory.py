"""The states of sequences that are cut into segments: a call may write them where it read them, as `linear_attention_packed` always does."""
import ctypes as C

import pytest
import torch

from tests.test_linear_attention import DTYPES, _decays, _rand

pytestmark = pytest.mark.gpu


def _operands(lens, N, D, dtype):
    T = sum(lens)
    q, k, v = (_rand(T, N, D, dtype=dtype, seed=s) for s in (1, 2, 3))
    return q, k, v, _decays(N, 6), torch.tensor([0] + lens).cumsum(0).int().cuda()


def _forward(ops, state_in, state_out):
    """acct_linear_fwd: (y, the workspace's states [slots, N, D, D])."""
    from acctransformer_b200 import _lib
    q, k, v, g, cu = ops
    a = _lib.LinearArgs()
    a.dtype = _lib.ACCT_BF16 if q.dtype == torch.bfloat16 else _lib.ACCT_F16
    a.B, (a.S, a.N, a.D), a.scale = cu.numel() - 1, q.shape, 0.125
    y = torch.empty_like(q)
    a.q, a.k, a.v, a.y, a.log_decay, a.cu_seqlens = (t.data_ptr() for t in (q, k, v, y, g, cu))
    a.state_in, a.state_out = (t.data_ptr() if t is not None else None for t in (state_in, state_out))
    a.workspace_bytes = _lib.load().acct_linear_fwd_workspace_bytes(C.byref(a))
    assert a.workspace_bytes > 0      # (cut)
    slots = torch.empty(a.workspace_bytes // (4 * a.N * a.D * a.D), a.N, a.D, a.D, device="cuda")
    a.workspace = slots.data_ptr()
    _lib.check(_lib.load().acct_linear_fwd(C.byref(a), C.c_void_p(torch.cuda.current_stream().cuda_stream)))
    return y, slots


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("lens,N,D", [([16384], 1, 64), ([8192], 2, 128), ([4097, 0, 6000], 1, 80)])
def test_in_place_and_apart_are_the_same(dt, lens, N, D):
    ops = _operands(lens, N, D, DTYPES[dt])
    state = _rand(len(lens), N, D, D, dtype=torch.float32, seed=4, scale=3.0)
    kept, after = state.clone(), torch.empty_like(state)
    y, _ = _forward(ops, state, after)
    assert torch.equal(state, kept)
    for _ in range(20):
        mine = state.clone()
        again, _ = _forward(ops, mine, mine)
        assert torch.equal(again, y) and torch.equal(mine, after)


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("N,D,T", [(1, 64, 16384), (2, 128, 5000)])
def test_first_segments_start_from_a_copy(dt, N, D, T):
    """No block of the launch that writes the states reads them where they were given: what is before the first segment lies in its slot."""
    ops = _operands([T], N, D, DTYPES[dt])
    state = _rand(1, N, D, D, dtype=torch.float32, seed=4)
    _, slots = _forward(ops, state, torch.empty_like(state))
    assert torch.equal(slots[0], state[0])
    # and states that are not given are zeros, whatever the slots held
    y, _ = _forward(ops, torch.zeros_like(state), torch.empty_like(state))
    none, _ = _forward(ops, None, torch.empty_like(state))
    assert torch.equal(y, none)
