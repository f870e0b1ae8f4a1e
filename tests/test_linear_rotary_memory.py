"""What the calls of linear attention and rotary positions write is no memory that they read as something else, views with gaps among it."""
import pytest
import torch

from tests.test_linear_attention import _decays, _ours

pytestmark = pytest.mark.gpu

T, N, D = 12, 2, 64


def _refused(call, *args, **more):
    with pytest.raises(ValueError, match="share memory"):
        call(*args, **more)


def _buffer(rows):
    """[rows, 3 N, D] with room behind: q, k, v are views with gaps."""
    buf = torch.zeros((rows * 3 * N + 64 * N) * D, dtype=torch.bfloat16, device="cuda")
    return buf, [t for t in buf[:rows * 3 * N * D].view(rows, 3 * N, D).split(N, 1)]


@pytest.mark.parametrize("at", [0, 1, 2, 5, 17, 3 * T - 1])
def test_out_among_the_rows_of_a_projection(at):
    """`out` begins `at` times N D values into the buffer: over rows, or over the end of them."""
    m = _ours()
    buf, (q, k, v) = _buffer(T)
    cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    out = buf[at * N * D:][:T * N * D].view(T, N, D)
    _refused(m.linear_attention_packed, q, k, v, _decays(N), cu, out=out)
    _refused(m.linear_attention_packed, q.clone(), k.clone(), v, _decays(N), cu, out=buf[(3 * T - 1) * N * D:][:T * N * D].view(T, N, D))
    behind = buf[3 * T * N * D:][:T * N * D].view(T, N, D)
    y, _ = m.linear_attention_packed(q, k, v, _decays(N), cu, out=behind)
    assert y.data_ptr() == behind.data_ptr()


def test_out_in_the_gaps():
    """Memory between the rows is other memory."""
    m = _ours()
    buf = torch.randn(2, 4, N, D, device="cuda").bfloat16()      # two sequences, and of each q, k, v and what is not read
    q, k, v = (buf[:, i].unsqueeze(2) for i in range(3))
    g = _decays(N)
    states = torch.zeros(2, 2, N, D, D, device="cuda")
    want = m.linear_attention_step(q[:1], k[:1], v[:1], g, states[0][:1])
    whole = m.linear_attention_step(q, k, v, g, states[1])
    assert torch.equal(m.linear_attention_step(q[:1], k[:1], v[:1], g, torch.zeros(1, N, D, D, device="cuda"), out=buf[0, 3].view(1, N, 1, D)), want)
    assert torch.equal(whole[:1], want)
    row = buf.view(-1, N, D)
    _refused(m.linear_attention_step, q, k, v, g, states[0], out=row[3:5].unsqueeze(2))      # the gap, and the next sequence's q


def test_state_among_the_rows():
    m = _ours()
    buf = torch.zeros(N * D * D * 4 + 4096, dtype=torch.bfloat16, device="cuda")
    state = buf[:N * D * D * 2].view(torch.float32).view(1, N, D, D)
    q, k, v = buf[N * D:][:3 * N * D * 8].view(8, 3 * N, D).split(N, 1)
    cu = torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    _refused(m.linear_attention_packed, q, k, v, _decays(N), cu, state=state)
    _refused(m.linear_attention_step, *(t[:1].unsqueeze(2) for t in (q, k, v)), _decays(N), state)


def test_rotary_in_place():
    rotary = _ours().Rotary(D)
    buf, (q, k, v) = _buffer(T)
    pos = torch.arange(T, device="cuda")
    rotary.apply_(q, k, pos)
    dense = buf[:T * N * D].view(T, N, D)
    _refused(rotary.apply_, dense, k, pos)
    _refused(rotary.apply_, k, dense, pos)
    _refused(rotary.apply_, q, q[:, :1], pos)
    for mine in (dense, q):
        at = mine[1].reshape(-1)[:2 * T].view(torch.int32) if mine is dense else buf[N * D - 2 * T:N * D].view(torch.int32)
        assert at.numel() == T and at.data_ptr() < dense.data_ptr() + dense.nbytes
        _refused(rotary.apply_, mine, None, at.copy_(pos))
        _refused(rotary.apply_, None, mine, at)
    rotary.apply_(q, buf[3 * T * N * D:][:T * N * D].view(T, N, D), pos)
