"""The backward's workspace: what the size query says is what the launch lays out, whatever surrounds the process."""
import glob
import os

import pytest

from acctransformer_b200 import _lib, build


def test_the_library_does_not_read_the_environment():
    """What a call computes, and how much memory has to be there for it, follows from its arguments: a variable of the process could
    make the size query and the launch disagree."""
    sources = glob.glob(os.path.join(build.CSRC, "*"))
    assert len(sources) > 20
    for path in sources:
        text = open(path).read()
        assert "getenv" not in text and "environ" not in text, path


@pytest.mark.parametrize("D, per_tile", [(8, 1), (64, 1), (128, 1), (136, 2), (160, 2), (256, 2)])
@pytest.mark.parametrize("S", [1, 128, 129, 8192])
def test_size(D, per_tile, S):
    """Row sums, turn counters (one per 128 query rows, two where halves of head_dim share them) and the work counter, fp32 dQ."""
    build.build()
    a = _lib.FaArgs()
    a.B, a.N, a.S_q, a.S_k, a.D = 2, 3, S, S, D
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    rest = up(6 * S * 4) + up((6 * -(-S // 128) * per_tile + 1) * 4)
    size = _lib.load().acct_fa_bwd_workspace_bytes
    assert size(a) == rest + 6 * S * D * 4
    a.flags = _lib.FLAG_GRAD_F32
    assert size(a) == rest
