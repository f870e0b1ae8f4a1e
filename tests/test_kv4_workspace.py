"""A decoding step without a workspace takes the memory that it can use, not that of the finest cut there is."""
import pytest
import torch

from acctransformer_b200 import _lib, build as _build


def _size(S, splits, weights=0, B=32, N=32, N_kv=8, D=128):
    _build.build()
    c = _lib.Kv4CacheArgs()
    c.B, c.N_kv, c.S_max, c.D = B, N_kv, S, D
    return _lib.load().acct_kv4_decode_workspace_bytes(c, N, splits, weights)


@pytest.mark.parametrize("S, most", [(1, 1), (512, 1), (513, 2), (5000, 10), (32768, 64), (1 << 20, 64), (2 ** 31 - 1, 64)])
def test_room_for_what_the_library_chooses(S, most):
    """Parts of a sequence are of 512 slots or more, and 64 at most."""
    assert _size(S, -1) == _size(S, most)
    assert _size(S, 0) == _size(S, 64)                       # calls with any number of parts
    if S < 1 << 20:
        assert _size(S, -1, 1) - _size(S, -1) == _size(S, 1, 1) - _size(S, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("S, lens", [(500, [500, 33]), (5000, [5000, 4097]), (40000, [40000, 3])])
@pytest.mark.parametrize("group", [1, 4, 12])
def test_a_step_without_a_workspace(S, lens, group):
    """Takes no more than that, and gives what a call with room for any cut does."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from acctransformer_b200 import Kv4Cache, Kv4Workspace
    B, N_kv, D = 2, 4, 128
    cache = Kv4Cache(B, N_kv, S, D)
    cache.append(*(torch.randn(B * S, N_kv, D, device="cuda").half() for _ in range(2)), torch.zeros(B, dtype=torch.int32, device="cuda"),
                 torch.tensor([0, S, 2 * S], dtype=torch.int32, device="cuda"))
    q, seq = torch.randn(B, N_kv * group, 1, D, device="cuda").half(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    for weights in (None, torch.zeros(B, N_kv, S, device="cuda")):
        room = Kv4Workspace(B, N_kv * group, N_kv, S, D, "cuda", weights=weights is not None)
        want = cache.decode(q, seq, weights=weights, workspace=room)
        del room
        torch.cuda.reset_peak_memory_stats()
        asked = lambda what: torch.cuda.memory_stats()[f"requested_bytes.all.{what}"]  # noqa: E731 (not what blocks they are given)
        before = asked("current")
        y = cache.decode(q, seq, weights=weights)
        taken = asked("peak") - before
        assert torch.equal(y, want)
        allowed = _size(S, min(64, -(-S // 512)), int(weights is not None), B, N_kv * group, N_kv, D)
        assert taken <= allowed + y.nbytes
