"""Linear attention and rotary positions as programs use them: neighbours that are not finite, views, streams, graphs, ranges of float16,
refusals that need a device."""
import pytest
import torch

from tests.test_linear_attention import DTYPES, _close, _decays, _ours, _rand, _state_close, attend

pytestmark = pytest.mark.gpu


def _packed(lens, N, N_kv, D, dtype, seed=0):
    T = sum(lens)
    q, k, v = (_rand(T, h, D, dtype=dtype, seed=seed + s) for s, h in ((1, N), (2, N_kv), (3, N_kv)))
    return q, k, v, _decays(N), torch.tensor([0] + lens).cumsum(0).int().cuda()


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("lens,N,D", [([100, 50, 200], 4, 128), ([7000, 7, 6500], 1, 64), ([130, 1, 127], 2, 40)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_sequences_do_not_see_their_neighbours(dt, lens, N, D, bad):
    m = _ours()
    q, k, v, g, cu = _packed(lens, N, N, D, DTYPES[dt])
    state = torch.randn(len(lens), N, D, D, device="cuda")
    want, s_want = m.linear_attention_packed(q, k, v, g, cu, state=state.clone())
    mine = slice(lens[0], lens[0] + lens[1])
    for t in (q, k, v):
        keep = t[mine].clone()
        t.fill_(bad)
        t[mine] = keep
    spoiled = state.clone()
    spoiled[0], spoiled[2] = bad, bad
    y, s = m.linear_attention_packed(q, k, v, g, cu, state=spoiled)
    assert torch.equal(y[mine], want[mine]) and torch.equal(s[1], s_want[1])


@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_padding_is_not_read(dt):
    m, lens = _ours(), [70, 0, 300, 129]
    B, N, N_kv, S, D = 4, 4, 2, 300, 96
    q, dy = (_rand(B, N, S, D, dtype=DTYPES[dt], seed=s) for s in (1, 2))
    k, v = (_rand(B, N_kv, S, D, dtype=DTYPES[dt], seed=s) for s in (3, 4))
    seq = torch.tensor(lens, device="cuda")
    outs = []
    for bad in (0.0, float("nan")):
        for b, n in enumerate(lens):
            for t in (q, k, v, dy):
                t[b, :, n:] = bad
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        y = m.linear_attention(*leaves, _decays(N), seq_lens=seq)
        outs.append((y.detach(),) + torch.autograd.grad(y, leaves, dy))
    assert all(torch.equal(a, b) and a.isfinite().all() for a, b in zip(*outs))
    # lengths out of range count as the nearest that is in it
    y = m.linear_attention(*(t.nan_to_num() for t in (q, k, v)), _decays(N), seq_lens=torch.tensor([70, -5, 4000, 129], device="cuda"))
    assert torch.equal(y, outs[0][0])


def test_rows_of_no_sequence_stay():
    m = _ours()
    q, k, v, g, _ = _packed([400], 2, 2, 64, torch.bfloat16)
    cu = torch.tensor([30, 200, 200, 333], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 7.0)
    y, _ = m.linear_attention_packed(q, k, v, g, cu, out=out)
    assert y.data_ptr() == out.data_ptr() and out[:30].eq(7.0).all() and out[333:].eq(7.0).all() and not out[30:333].eq(7.0).any(-1).all()
    # nothing at all
    none, s = m.linear_attention_packed(q[:0], k[:0], v[:0], g, torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert none.shape == (0, 2, 64) and s.eq(0).all()
    s = torch.randn(2, 2, 64, 64, device="cuda")
    before = s.clone()
    m.linear_attention_packed(q[:0], k[:0], v[:0], g, torch.zeros(3, dtype=torch.int32, device="cuda"), state=s)
    assert torch.equal(s, before)


@pytest.mark.parametrize("B", [65, 300])
def test_many_sequences(B):
    m = _ours()
    lens = [(37 * b) % 150 for b in range(B)]
    q, k, v, g, cu = _packed(lens, 2, 1, 64, torch.float16)
    y, s = m.linear_attention_packed(q, k, v, g, cu)
    for b in (0, 1, B // 2, B - 1):
        n, at = lens[b], sum(lens[:b])
        y1, s1 = m.linear_attention_packed(q[at:at + n], k[at:at + n], v[at:at + n], g, torch.tensor([0, n], dtype=torch.int32, device="cuda"))
        assert torch.equal(y[at:at + n], y1) and torch.equal(s[b], s1[0])


@pytest.mark.parametrize("dt", sorted(DTYPES))
def test_views(dt):
    """[B, S, heads, D] behind one projection, and addresses that are no multiple of 16 bytes, give the same bits."""
    m, dtype = _ours(), DTYPES[dt]
    B, N, N_kv, S, D = 2, 4, 2, 200, 64
    qkv = _rand(B, S, N + 2 * N_kv, D, dtype=dtype, seed=1)
    parts = [t.transpose(1, 2) for t in qkv.split([N, N_kv, N_kv], 2)]
    g, dy = _decays(N), _rand(B, S, N, D, dtype=dtype, seed=2).transpose(1, 2)

    def run(ops, d):
        leaves = [t.detach().requires_grad_() for t in ops]
        y = m.linear_attention(*leaves, g)
        return (y.detach(),) + torch.autograd.grad(y, leaves, d)
    want = run([t.contiguous() for t in parts], dy.contiguous())

    def shifted(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        buf[1:] = t.reshape(-1)
        return buf[1:].view(t.shape)
    for ops, d in ((parts, dy), ([shifted(t) for t in parts], shifted(dy)), ([t.contiguous() for t in parts], dy.expand_as(dy))):
        assert all(torch.equal(a, b) for a, b in zip(run(ops, d), want))
    rows = [t[0] for t in qkv.split([N, N_kv, N_kv], 2)]
    cu = torch.tensor([0, 120, S], dtype=torch.int64, device="cuda")
    w = m.linear_attention_packed(*(t.contiguous() for t in rows), g, cu)
    for ops in (rows, [shifted(t) for t in rows]):
        assert all(torch.equal(a, b) for a, b in zip(m.linear_attention_packed(*ops, g.double(), cu), w))
    s1, s2 = torch.zeros(2, B, N, D, D, device="cuda")
    one = [t[:, :, 5:6] for t in parts]
    assert torch.equal(m.linear_attention_step(*one, g, s1), m.linear_attention_step(*(shifted(t) for t in one), g, s2)) and torch.equal(s1, s2)


@pytest.mark.parametrize("size_q,size_k,size_v", [(300.0, 300.0, 1e-3), (1e-3, 1e-3, 300.0), (1e-4, 100.0, 1.0), (1.0, 1e-4, 1e-4)])
def test_float16_keeps_its_bits_at_any_size(size_q, size_k, size_v):
    """Scores past the largest float16, weighted values and states below the smallest normal one: the rounding of the output, and of the
    scores and states in between, is that of values near 1."""
    m, D, n = _ours(), 64, 300
    q, k, v = (_rand(n, 2, D, dtype=torch.float16, seed=s, scale=size) for s, size in ((1, size_q), (2, size_k), (3, size_v)))
    g = torch.tensor([-0.02, -3.0], device="cuda")
    scale = 1.0 / (size_q * size_k * size_v)
    y, state = m.linear_attention_packed(q, k, v, g, torch.tensor([0, n], dtype=torch.int32, device="cuda"), scale=scale)
    x = [t.transpose(0, 1) for t in (q, k, v)]
    want, s1 = attend(*x, g)
    most, s_most = attend(*(t.abs() for t in x), g)
    _close(y.transpose(0, 1), want * scale, most * scale, torch.float16, n + 2 * D)
    # values far below the largest of their chunk keep fewer bits: by the chunk's largest value, 2^-36
    _state_close(state[0], s1, s_most + s_most.amax() * 2.0 ** -12, 140)


def test_steps_follow_their_decay():
    """A decay near 1 is multiplied with the state thousands of times: an error of a rounding each time would add up to 10^-4."""
    m, D = _ours(), 16
    g = torch.tensor([-1e-4, -3e-3], device="cuda")
    state = torch.full((1, 2, D, D), 1.0, device="cuda")
    zero, steps = torch.zeros(1, 2, 1, D, device="cuda", dtype=torch.bfloat16), 4000
    for _ in range(steps):
        m.linear_attention_step(zero, zero, zero, g, state)
    want = torch.exp(g.double() * steps)
    # 4 000 roundings of the state, of either sign or at worst all of one: 4000 2^-24
    assert ((state[0, :, 0, 0].double() - want).abs() <= want * steps * 2.0 ** -24 + 2.0 ** -126).all()
    n = 40000      # and in chunks: two roundings in each
    rows = torch.zeros(n, 2, D, device="cuda", dtype=torch.bfloat16)
    state = torch.full((1, 2, D, D), 1.0, device="cuda")
    m.linear_attention_packed(rows, rows, rows, g, torch.tensor([0, n], dtype=torch.int32, device="cuda"), state=state)
    want = torch.exp(g.double() * n)
    # (exp(-120) = 8 10^-53 is less than the smallest number of float32)
    assert ((state[0, :, 0, 0].double() - want).abs() <= want * (2 * n / 128 + 8) * 2.0 ** -23 + 2.0 ** -126).all()


def test_same_bits_every_time():
    m = _ours()
    B, N, N_kv, S, D = 2, 8, 2, 1500, 64
    q, dy = (_rand(B, N, S, D, dtype=torch.bfloat16, seed=s) for s in (1, 2))
    k, v = (_rand(B, N_kv, S, D, dtype=torch.bfloat16, seed=s) for s in (3, 4))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    runs = []
    for _ in range(3):
        y = m.linear_attention(*leaves, _decays(N))
        runs.append((y.detach(),) + torch.autograd.grad(y, leaves, dy))
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))


def test_captured_prompts_and_steps():
    m, N, D = _ours(), 4, 64
    rotary = m.Rotary(D, (8, 12, 12))
    q, k, v, g, cu = _packed([150, 40, 210], N, 2, D, torch.bfloat16)
    pos = torch.randint(0, 100, (3, 400), dtype=torch.int32, device="cuda")
    state = torch.zeros(3, N, D, D, device="cuda")
    one = [t[:3].unsqueeze(2) for t in (q, k, v)]

    def run():
        a, b = rotary(q, k, pos)
        y, _ = m.linear_attention_packed(a, b, v, g, cu, state=state)
        return y, m.linear_attention_step(*one, g, state)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, z = run()
    for seed, lens in ((5, [150, 40, 210]), (6, [0, 399, 1]), (7, [128, 128, 100])):
        for t, s in ((q, 1), (k, 2), (v, 3)):
            t.copy_(_rand(*t.shape, dtype=t.dtype, seed=seed + s))
        pos.random_(0, 1000)
        cu.copy_(torch.tensor([0] + lens).cumsum(0))
        state.normal_()
        before = state.clone()
        graph.replay()
        got = y.clone(), z.clone(), state.clone()
        state.copy_(before)
        want = run() + (state,)
        n = sum(lens)
        assert torch.equal(got[0][:n], want[0][:n]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])


def test_captured_training_while_an_eager_graph_lives():
    m = _ours()
    B, N, S, D = 1, 2, 300, 64
    cell = m.LinearAttention(N, D, rotary=m.Rotary(D)).cuda()
    leaves = [_rand(B, N, S, D, dtype=torch.bfloat16, seed=s).requires_grad_() for s in (1, 2, 3)]
    dy = _rand(B, N, S, D, dtype=torch.bfloat16, seed=4)
    pos = torch.arange(S, dtype=torch.int32, device="cuda")
    # (on the stream of the capture: autograd joins a leaf's stream, and a capture cannot be joined with another one)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = cell(*leaves, positions=pos)      # stays alive over the capture
        torch.autograd.grad(cell(*leaves, positions=pos), leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = cell(*leaves, positions=pos)
        grads = torch.autograd.grad(y, leaves, dy)
    graph.replay()
    want = torch.autograd.grad(eager, leaves, dy)
    assert torch.equal(y, eager) and all(torch.equal(a, b) for a, b in zip(grads, want))


def test_other_streams():
    m = _ours()
    q, k, v, g, cu = _packed([700, 300], 4, 4, 128, torch.bfloat16)
    want = m.linear_attention_packed(q, k, v, g, cu)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:      # at once
        with torch.cuda.stream(s):
            outs.append(m.linear_attention_packed(q, k, v, g, cu))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))


@pytest.mark.parametrize("N,T", [(1, 40000), (16, 300)])
def test_starts_that_are_no_starts(N, T):
    """Rows that two sequences claim, starts that go back or leave the rows: nothing outside the outputs is touched."""
    m, D = _ours(), 64
    q, k, v = (_rand(T, N, D, dtype=torch.bfloat16, seed=s) for s in (1, 2, 3))
    g = _decays(N, 6)
    good = torch.tensor([0, T // 3, T], dtype=torch.int32, device="cuda")
    want = m.linear_attention_packed(q, k, v, g, good)
    for cu in ([0, T, 0, T, 0, T], [-5, T + 1000, 7, 3, 2 ** 31 - 1], [T, T - 1, 5, -2 ** 31], [0, 2 ** 31 - 1, -1, T]):
        band = torch.full((3, T, N, D), 7.0, device="cuda", dtype=torch.bfloat16)
        y, state = m.linear_attention_packed(q, k, v, g, torch.tensor(cu, dtype=torch.int32, device="cuda"), out=band[1])
        torch.cuda.synchronize()
        assert band[0].eq(7.0).all() and band[2].eq(7.0).all() and state.shape[0] == len(cu) - 1
    assert all(torch.equal(a, b) for a, b in zip(m.linear_attention_packed(q, k, v, g, good), want))
    from acctransformer_b200 import _lib
    _lib.device_status()


def test_inference_mode_and_casts():
    m, N, D = _ours(), 4, 64
    cell = m.LinearAttention(N, D, log_decay=[-0.1, -0.0123456, 0.0, -3.0], rotary=m.Rotary(D, (16, 16)))
    assert cell.cuda().bfloat16().log_decay.dtype == torch.float32 and cell.log_decay.is_cuda
    q, k, v = (_rand(2, N, 200, D, dtype=torch.bfloat16, seed=s) for s in (1, 2, 3))
    want = cell(q, k, v)
    with torch.inference_mode():
        a, b, c = (t.clone() for t in (q, k, v))
        assert torch.equal(cell(a, b, c), want)
        state = torch.zeros(2, N, D, D, device="cuda")
        cell.step(*(t[:, :, :1] for t in (a, b, c)), state, positions=torch.zeros(2, 2, 1, dtype=torch.int32, device="cuda"))
        assert state.ne(0).any()


def test_refusals():
    m = _ours()
    q, k, v, g, cu = _packed([64], 4, 2, 64, torch.bfloat16)
    state = torch.zeros(1, 4, 64, 64, device="cuda")
    call = m.linear_attention_packed
    for bad in ((q.float(), k, v, g, cu), (q, k.half(), v, g, cu), (q, k[:-1], v[:-1], g, cu), (q, k[..., :32], v[..., :32], g, cu), (q, k, v, g[:3], cu), (q, k, v, g.int(), cu),
                (q, k, v, g, cu[:1]), (q, k, v, g, cu.float()), (q, k, v, g, cu.cpu()), (q, k, v, g.cpu(), cu), (q[:, :3], k, v, g[:3], cu), (q.cpu(), k, v, g, cu)):
        with pytest.raises(ValueError):
            call(*bad)
    for bad in (state.half(), state[:, :3], state.transpose(2, 3), torch.zeros(2, 4, 64, 64, device="cuda"), state.cpu()):
        with pytest.raises(ValueError):
            call(q, k, v, g, cu, state=bad)
    with pytest.raises(ValueError, match="share memory"):
        call(q, k, v, g, cu, out=q)
    with pytest.raises(ValueError):
        call(q, k, v, g, cu, out=q.half())
    one = [t[:1].unsqueeze(2) for t in (q, k, v)]
    with pytest.raises(ValueError, match="one token"):
        m.linear_attention_step(*(t[:2].unsqueeze(0).transpose(1, 2) for t in (q, k, v)), g, state)
    with pytest.raises(ValueError, match="share memory"):
        m.linear_attention_step(*one, g, state, out=state.view(torch.bfloat16).view(-1)[:256].view(1, 4, 1, 64))
    with pytest.raises(ValueError, match="log_decay has no gradient"):
        call(q, k, v, g.clone().requires_grad_(), cu)
    wide = [torch.zeros(1, 1, 8, 136, device="cuda", dtype=torch.float16) for _ in range(3)]
    from acctransformer_b200._lib import AcctError
    with pytest.raises(AcctError, match="head_dim"):
        m.linear_attention(*wide, g[:1])
    leaves = [t.requires_grad_() for t in (torch.randn(1, 2, 9, 64, device="cuda").half() for _ in range(3))]
    y = m.linear_attention(*leaves, g[:2])
    (dq,) = torch.autograd.grad(y.sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        dq.sum().backward()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.sum(), leaves[1])
    lens = torch.tensor([9], dtype=torch.int32, device="cuda")
    y = m.linear_attention(*leaves, g[:2], seq_lens=lens)
    lens.fill_(3)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_rotary_views_and_refusals():
    m = _ours()
    T, N, N_kv, D = 50, 4, 2, 64
    rotary = m.Rotary(D, (16, 16))
    qkv = _rand(T, N + 2 * N_kv, D, dtype=torch.float16, seed=1)
    pos = torch.randint(0, 99, (2, T), device="cuda")
    q, k, v = qkv.split([N, N_kv, N_kv], 1)
    want, kept = rotary(q.contiguous(), k.contiguous(), pos), v.clone()
    assert all(torch.equal(a, b) for a, b in zip(rotary(q, k, pos), want))
    version = qkv._version
    rotary.apply_(q, k, pos)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, kept) and qkv._version > version
    x = _rand(3, N, T, D, dtype=torch.bfloat16, seed=2)
    xt = x.transpose(1, 2).contiguous().transpose(1, 2)
    shared = rotary(x, None, pos)[0]
    assert torch.equal(rotary(xt, None, pos)[0], shared) and torch.equal(rotary(x, None, pos.unsqueeze(1).expand(2, 3, T))[0], shared)
    assert rotary(q[:0], k[:0], pos[:, :0])[0].shape == (0, N, D)
    for bad in ((q, k, pos[:1]), (q, k[:-1], pos), (q, k, pos.float()), (q.float(), k.float(), pos), (q[..., :32], k[..., :32], pos), (q, k, pos.cpu()), (None, None, pos),
                (x, None, pos.unsqueeze(1).expand(2, 2, T)), (q, k.bfloat16(), pos)):
        with pytest.raises(ValueError):
            rotary(*bad)
    with pytest.raises(ValueError, match="share memory"):
        rotary.apply_(q, q, pos)
    buf = torch.zeros(T * N * D + 1, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="16 bytes"):
        rotary.apply_(buf[1:].view(T, N, D), None, pos)
    leaf = _rand(T, N, D, dtype=torch.float16, seed=3).requires_grad_()
    with pytest.raises(ValueError, match="has no gradient"):
        rotary.apply_(leaf, None, pos)
    # a turn is linear: its second derivative is the turn again, and turning back gives the values again
    y = rotary(leaf, None, pos)[0]
    (back,) = torch.autograd.grad(y, leaf, y, create_graph=True)
    # turned twice, rounded twice: each of the four products of a pair's length, 2^-11 each time
    assert ((back - leaf).abs() <= 4 * 2.0 ** -11 * (leaf.abs().amax() * 1.5)).all()
    (again,) = torch.autograd.grad(back, y, torch.ones_like(back))
    assert again.isfinite().all()
    pos2 = pos.int()
    y = rotary(leaf, None, pos2)[0]
    pos2.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
