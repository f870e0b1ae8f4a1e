"""Linear attention with a decay for each head on the GPU against its definition in 64 bits: batches and their gradients, packed prompts
with states, single tokens, and all of them in a row.

Tolerances.  The 16-bit output is rounded once: at most u = eps / 2 of the value.  What the products round to 16 bits on their way
(the weighted scores, the state that queries read; the weighted rows that go into a state keep 16 bits and more) is off by at most
u of each term of a sum, so an output is off by at most u (|y| + 2 A), A the same sum over absolute values, and by fp32 sums' n 2^-24 A
besides.  The errors of many terms do not all have one sign, so that bound is loose; it needs no other assumption."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _ours():
    import acctransformer_b200 as m
    return m


def attend(q, k, v, g, state=None, reverse=False, chunk=64):
    """[N, n, D] in float64: outputs and the state behind; the recurrence, `chunk` tokens at a time."""
    N, n, D = q.shape
    g = g.double()
    state = torch.zeros(N, D, D, dtype=torch.float64, device=q.device) if state is None else state.double()
    out = []
    for at in range(0, n, chunk):
        x, y, z = (t[:, at:at + chunk].double() for t in (q, k, v))
        m = x.shape[1]
        i = torch.arange(m, dtype=torch.float64, device=q.device)
        w = torch.exp(g[:, None, None] * (i[:, None] - i).clamp_min(0)).tril()
        out.append((x @ y.transpose(-1, -2) * w) @ z + torch.exp(g[:, None] * (i + 1))[..., None] * (x @ state))
        state = torch.exp(g * m)[:, None, None] * state + (y * torch.exp(g[:, None] * (m - 1 - i))[..., None]).transpose(-1, -2) @ z
    return (torch.cat(out, 1) if out else torch.zeros(N, 0, D, dtype=torch.float64, device=q.device)), state


def _rand(*shape, dtype, seed, scale=1.0, shift=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=gen) * scale + shift).to(dtype)


def _decays(N, seed=0):
    """From no decay at all to one that leaves nothing of the token before."""
    some = [0.0, -1e-4, -0.01, -0.3, -2.0, -120.0, -0.07, -0.002]
    return torch.tensor([some[(h + seed) % len(some)] for h in range(N)], device="cuda")


def _close(got, want, most, dtype, terms):
    """|got - want| against u (|want| + 2 A) + terms 2^-24 A, A = `most`."""
    u = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny
    bound = u * (want.abs() + 2 * most) + terms * 2.0 ** -24 * most + tiny
    err = (got.double() - want).abs()
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"off by {worst:.2f} of the bound"


def _state_close(got, want, most, terms):
    # fp32 throughout: products exact or rounded to 22 bits and more, `terms` additions
    bound = (terms + 16) * 2.0 ** -23 * most + 1e-30
    worst = ((got.double() - want).abs() / bound).max().item()
    assert worst <= 1.0, f"off by {worst:.2f} of the bound"


def _heads(x, N):
    """[N_kv, ...] -> [N, ...]"""
    return x.repeat_interleave(N // x.shape[0], 0)


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("lens,N,N_kv,D", [
    ([1], 1, 1, 64), ([5, 0, 128, 129], 4, 4, 128), ([127, 1, 300], 8, 2, 64), ([77, 513], 3, 1, 80), ([1000, 2, 384, 640, 0], 6, 6, 128),
    ([200] * 9, 2, 2, 40), ([2500], 8, 4, 128), ([31, 33, 64], 16, 16, 8), ([1500, 1500], 2, 2, 96), ([4000], 1, 1, 120)])
@pytest.mark.parametrize("with_state", [False, True])
def test_packed(dt, lens, N, N_kv, D, with_state):
    dtype = DTYPES[dt]
    T = sum(lens)
    q, k, v = (_rand(T, h, D, dtype=dtype, seed=s, shift=0.1 * s) for s, h in ((1, N), (2, N_kv), (3, N_kv)))
    g = _decays(N)
    cu = torch.tensor([0] + lens).cumsum(0).int().cuda()
    state = _rand(len(lens), N, D, D, dtype=torch.float32, seed=4, scale=3.0) if with_state else None
    before = state.clone() if with_state else None
    y, after = _ours().linear_attention_packed(q, k, v, g, cu, state=state)
    if with_state:
        assert after is state or after.data_ptr() == state.data_ptr()
    scale, at = D ** -0.5, 0
    for b, n in enumerate(lens):
        x = [t[at:at + n].double().transpose(0, 1) for t in (q, k, v)]
        x[1], x[2] = _heads(x[1], N), _heads(x[2], N)
        s0 = before[b] if with_state else None
        want, s1 = attend(*x, g, s0)
        most, s_most = attend(*(t.abs() for t in x), g, None if s0 is None else s0.abs())
        _close(y[at:at + n].transpose(0, 1), want * scale, most * scale, dtype, n + 2 * D)
        _state_close(after[b], s1, s_most, min(n, 128) + n // 128)
        at += n


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("B,N,N_kv,S,D,lens", [
    (1, 1, 1, 1, 64, None), (2, 4, 4, 130, 128, None), (3, 8, 2, 257, 64, [257, 0, 100]), (1, 3, 1, 500, 80, None), (2, 2, 2, 1024, 128, [1, 900]),
    (2, 6, 6, 384, 40, None), (1, 8, 8, 2100, 128, None), (5, 4, 1, 127, 96, [127, 126, 64, 3, 0])])
def test_training(dt, B, N, N_kv, S, D, lens):
    dtype = DTYPES[dt]
    q, dy = (_rand(B, N, S, D, dtype=dtype, seed=s) for s in (1, 2))
    k, v = (_rand(B, N_kv, S, D, dtype=dtype, seed=s, shift=0.2) for s in (3, 4))
    g = _decays(N, 1)
    seq = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_() for t in (q, k, v)]
    y = _ours().linear_attention(q, k, v, g, seq_lens=seq)
    grads = torch.autograd.grad(y, leaves, dy)
    scale = D ** -0.5
    for b in range(B):
        n = S if lens is None else lens[b]
        for t in (y,) + grads:
            assert t[b, :, n:].eq(0).all()
        xq, xd = q[b, :, :n].detach().double(), dy[b, :, :n].double()
        xk, xv = (_heads(t[b, :, :n].detach().double(), N) for t in (k, v))
        flip = lambda t: t.flip(1)  # noqa: E731
        pairs = [(y[b, :, :n], (xq, xk, xv), False, False), (grads[0][b, :, :n], (xd, xv, xk), False, False),
                 (grads[1][b, :, :n], (xv, xd, xq), True, True), (grads[2][b, :, :n], (xk, xq, xd), True, True)]
        for got, ops, back, shared in pairs:
            ops = [flip(t) for t in ops] if back else ops
            want, most = attend(*ops, g)[0], attend(*(t.abs() for t in ops), g)[0]
            if back:
                want, most = flip(want), flip(most)
            if shared:
                want, most = (t.unflatten(0, (N_kv, -1)).sum(1) for t in (want, most))
            _close(got, want * scale, most * scale, dtype, n + 2 * D)


def test_gradient_against_differences():
    """The formula's gradients, by which the kernels are judged above, against differences of the definition."""
    torch.manual_seed(0)
    N, n, D = 2, 7, 8
    g = torch.tensor([-0.3, -0.01], device="cuda", dtype=torch.float64)
    x = [torch.randn(N, n, D, device="cuda", dtype=torch.float64) for _ in range(4)]
    f = lambda q, k, v: (attend(q, k, v, g)[0] * x[3]).sum()  # noqa: E731
    formula = [attend(x[3], x[2], x[1], g)[0], attend(x[2].flip(1), x[3].flip(1), x[0].flip(1), g)[0].flip(1),
               attend(x[1].flip(1), x[0].flip(1), x[3].flip(1), g)[0].flip(1)]
    for i in range(3):
        for at in ((0, 0, 0), (1, 3, 5), (0, 6, 7)):
            h = 1e-6
            up, down = [t.clone() for t in x[:3]], [t.clone() for t in x[:3]]
            up[i][at] += h
            down[i][at] -= h
            assert abs((f(*up) - f(*down)) / (2 * h) - formula[i][at]) < 1e-7


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("B,N,N_kv,D", [(1, 1, 1, 64), (4, 32, 8, 128), (7, 12, 3, 80), (3, 2, 2, 8), (2, 5, 5, 120)])
def test_step(dt, B, N, N_kv, D):
    dtype = DTYPES[dt]
    q, k, v = (_rand(B, h, 1, D, dtype=dtype, seed=s) for s, h in ((1, N), (2, N_kv), (3, N_kv)))
    g = _decays(N)
    state = _rand(B, N, D, D, dtype=torch.float32, seed=4)
    before = state.double()
    y = _ours().linear_attention_step(q, k, v, g, state)
    xk, xv = (t.double().repeat_interleave(N // N_kv, 1) for t in (k, v))
    want = before * torch.exp(g.double())[:, None, None] + xk.transpose(-1, -2) * xv
    most = before.abs() * torch.exp(g.double())[:, None, None] + (xk.transpose(-1, -2) * xv).abs()
    _state_close(state, want, most, 2)
    _close(y, q.double() @ want * D ** -0.5, q.double().abs() @ most * D ** -0.5, dtype, D)


@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_prompts_then_tokens_then_prompts(dt):
    """As a server uses them, rotary positions included: the pieces give what one call over everything gives."""
    m, dtype = _ours(), DTYPES[dt]
    N, N_kv, D, lens, more = 4, 2, 64, [150, 3, 260], 5
    cell = m.LinearAttention(N, D, rotary=m.Rotary(D, (8, 12, 12))).cuda()
    B, S = len(lens), max(lens) + 2 * more
    q, k, v = (_rand(B, h, S, D, dtype=dtype, seed=s) for s, h in ((1, N), (2, N_kv), (3, N_kv)))
    pos = torch.randint(0, 500, (3, B, S), device="cuda", dtype=torch.int32)
    whole = cell(q, k, v, seq_lens=torch.tensor([n + 2 * more for n in lens], dtype=torch.int32, device="cuda"), positions=pos)
    rq, rk = cell.rotary(q, k, pos)
    A = torch.stack([attend(rq[b].abs(), _heads(rk[b].abs(), N), _heads(v[b].abs(), N), cell.log_decay)[0] for b in range(B)]) * D ** -0.5

    def packed(t, a, n):
        return torch.cat([t[b, :, a[b]:a[b] + n[b]].transpose(0, 1) for b in range(B)])

    def check(y, a, n, rows):
        want, most = packed(whole.double(), a, n), packed(A, a, n)
        _close(y, want, most + want.abs(), dtype, 2 * rows)      # (both are rounded)

    def prompt(a, n, state):
        cu = torch.tensor([0] + n).cumsum(0).int().cuda()
        p = torch.cat([pos[:, b, a[b]:a[b] + n[b]] for b in range(B)], 1)
        y, state = cell.prompt(*(packed(t, a, n) for t in (q, k, v)), cu, state=state, positions=p)
        check(y, a, n, S)
        return state

    at = [0] * B
    state = prompt(at, lens, None)
    at = list(lens)
    for _ in range(more):
        one = lambda t: torch.stack([t[b, :, at[b]:at[b] + 1] for b in range(B)])  # noqa: E731
        y = cell.step(one(q), one(k), one(v), state, positions=torch.stack([pos[:, b, at[b]:at[b] + 1] for b in range(B)], 1))
        check(y.squeeze(2), at, [1] * B, S)
        at = [x + 1 for x in at]
    prompt(at, [more] * B, state)
