"""Linear attention where there are few heads: long sequences are cut into segments, whose states are found first and joined."""
import pytest
import torch

from tests.test_linear_attention import DTYPES, _close, _decays, _heads, _ours, _rand, _state_close, attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("lens,N,N_kv,D", [
    ([3000], 2, 2, 128), ([128 * 16], 1, 1, 64), ([2500, 0, 1, 4097, 640], 2, 1, 80), ([0, 9000, 127], 1, 1, 128), ([1, 5000], 4, 2, 40)])
@pytest.mark.parametrize("with_state", [False, True])
def test_packed(dt, lens, N, N_kv, D, with_state):
    dtype = DTYPES[dt]
    T = sum(lens)
    q, k, v = (_rand(T, h, D, dtype=dtype, seed=s) for s, h in ((1, N), (2, N_kv), (3, N_kv)))
    g = _decays(N, 6)      # slow ones, which carry a state over segments
    cu = torch.tensor([0] + lens).cumsum(0).int().cuda()
    state = _rand(len(lens), N, D, D, dtype=torch.float32, seed=4, scale=3.0) if with_state else None
    before = state.clone() if with_state else None
    y, after = _ours().linear_attention_packed(q, k, v, g, cu, state=state)
    scale, at = D ** -0.5, 0
    for b, n in enumerate(lens):
        x = [t[at:at + n].double().transpose(0, 1) for t in (q, k, v)]
        x[1], x[2] = _heads(x[1], N), _heads(x[2], N)
        s0 = before[b] if with_state else None
        want, s1 = attend(*x, g, s0)
        most, s_most = attend(*(t.abs() for t in x), g, None if s0 is None else s0.abs())
        _close(y[at:at + n].transpose(0, 1), want * scale, most * scale, dtype, n + 2 * D)
        _state_close(after[b], s1, s_most, min(n, 128) + n // 128 + 64)
        at += n


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("B,N,N_kv,S,D,lens", [(1, 1, 1, 5000, 128, None), (2, 2, 1, 2177, 64, [2177, 300]), (1, 3, 3, 4096, 96, None), (3, 1, 1, 3001, 128, [0, 3001, 2000])])
def test_training(dt, B, N, N_kv, S, D, lens):
    dtype = DTYPES[dt]
    q, dy = (_rand(B, N, S, D, dtype=dtype, seed=s) for s in (1, 2))
    k, v = (_rand(B, N_kv, S, D, dtype=dtype, seed=s) for s in (3, 4))
    g = _decays(N, 6)
    seq = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_() for t in (q, k, v)]
    y = _ours().linear_attention(q, k, v, g, seq_lens=seq)
    grads = torch.autograd.grad(y, leaves, dy)
    scale = D ** -0.5
    flip = lambda t: t.flip(1)  # noqa: E731
    for b in range(B):
        n = S if lens is None else lens[b]
        xq, xd = q[b, :, :n].detach().double(), dy[b, :, :n].double()
        xk, xv = (_heads(t[b, :, :n].detach().double(), N) for t in (k, v))
        for got, ops, back, shared in [(y, (xq, xk, xv), False, False), (grads[0], (xd, xv, xk), False, False),
                                       (grads[1], (xv, xd, xq), True, True), (grads[2], (xk, xq, xd), True, True)]:
            ops = [flip(t) for t in ops] if back else ops
            want, most = attend(*ops, g)[0], attend(*(t.abs() for t in ops), g)[0]
            if back:
                want, most = flip(want), flip(most)
            if shared:
                want, most = (t.unflatten(0, (N_kv, -1)).sum(1) for t in (want, most))
            _close(got[b, :, :n], want * scale, most * scale, dtype, n + 2 * D)
            assert got[b, :, n:].eq(0).all()
