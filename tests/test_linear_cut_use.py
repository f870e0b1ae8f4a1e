"""Sequences that are cut into segments, three launches and a workspace, as programs use them: again, on several streams at once, captured and
replayed on other operands, captured twice."""
import ctypes as C

import pytest
import torch

from tests.test_linear_attention import DTYPES, _decays, _ours, _rand

pytestmark = pytest.mark.gpu

SIZES = [([16384], 1, 1, 64), ([8000, 3, 5000], 2, 1, 128)]


def _is_cut(B, N, S, D, backward=False):
    from acctransformer_b200 import _lib
    a = _lib.LinearArgs()
    a.B, a.N, a.S, a.D = B, N, S, D
    a.cu_seqlens = None if backward else 4096      # (not read)
    lib = _lib.load()
    return (lib.acct_linear_bwd_workspace_bytes if backward else lib.acct_linear_fwd_workspace_bytes)(C.byref(a)) > 0


def _operands(lens, N, N_kv, D, dtype, seed):
    T = sum(lens)
    q, k, v = (_rand(T, h, D, dtype=dtype, seed=10 * seed + s) for s, h in ((1, N), (2, N_kv), (3, N_kv)))
    state = _rand(len(lens), N, D, D, dtype=torch.float32, seed=10 * seed + 4, scale=2.0)
    return q, k, v, _decays(N, 6), torch.tensor([0] + lens).cumsum(0).int().cuda(), state


def _run(ops):
    q, k, v, g, cu, state = ops
    return _ours().linear_attention_packed(q, k, v, g, cu, state=state)


def _same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("lens,N,N_kv,D", SIZES)
def test_same_bits_every_time(dt, lens, N, N_kv, D):
    assert _is_cut(len(lens), N, sum(lens), D)
    ops = _operands(lens, N, N_kv, D, DTYPES[dt], 1)
    runs = [_run(ops[:5] + (ops[5].clone(),)) for _ in range(10)]
    assert all(_same(r, runs[0]) for r in runs[1:])


@pytest.mark.parametrize("lens,N,N_kv,D", SIZES)
def test_streams_at_once(lens, N, N_kv, D):
    """Different operands on every stream: memory that calls shared would show."""
    assert _is_cut(len(lens), N, sum(lens), D)
    ops = [_operands(lens, N, N_kv, D, torch.bfloat16, i) for i in range(4)]
    want = [_run(o[:5] + (o[5].clone(),)) for o in ops]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ops]
    for _ in range(5):
        outs, states = [], [o[5].clone() for o in ops]
        torch.cuda.synchronize()
        for o, state, s in zip(ops, states, streams):
            with torch.cuda.stream(s):
                outs.append(_run(o[:5] + (state,)))
        torch.cuda.synchronize()
        assert all(_same(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("lens,N,N_kv,D", SIZES)
def test_two_graphs(lens, N, N_kv, D):
    """Captured with operands of their own, replayed in turn on others, the second one while the first one's results are kept."""
    ops = [_operands(lens, N, N_kv, D, torch.float16, i) for i in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for o in ops:
            _run(o)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for o in ops:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(_run(o))
    T = sum(lens)
    for seed, n in ((5, lens), (6, [T - 1] + [0] * (len(lens) - 2) + [1] if len(lens) > 1 else lens), (7, lens)):
        before = []
        for i, o in enumerate(ops):
            for t, x in zip(o[:3], _operands(lens, N, N_kv, D, torch.float16, seed + 10 * i)):
                t.copy_(x)
            o[4].copy_(torch.tensor([0] + n).cumsum(0))
            o[5].normal_()
            before.append(o[5].clone())
        for graph in graphs:
            graph.replay()
        got = [(y.clone(), s.clone()) for y, s in outs]
        for o, state, g in zip(ops, before, got):
            want = _run(o[:5] + (state,))
            assert _same(g, want)


@pytest.mark.parametrize("B,N,N_kv,S,D", [(1, 1, 1, 8001, 64), (2, 2, 1, 5000, 128)])
def test_gradients(B, N, N_kv, S, D):
    """Again, on streams at once, and from a graph."""
    assert _is_cut(B, N, S, D) and _is_cut(B, N, S, D, backward=True)
    m, g = _ours(), _decays(N, 6)
    sets = []
    for i in range(3):
        leaves = [_rand(B, h, S, D, dtype=torch.bfloat16, seed=10 * i + s).requires_grad_() for s, h in ((1, N), (2, N_kv), (3, N_kv))]
        sets.append((leaves, _rand(B, N, S, D, dtype=torch.bfloat16, seed=10 * i + 4)))

    def run(leaves, d):
        y = m.linear_attention(*leaves, g)
        return (y.detach(),) + torch.autograd.grad(y, leaves, d)
    want = [run(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        outs = []
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                outs.append(run(*s))
        torch.cuda.synchronize()
        assert all(_same(a, b) for a, b in zip(outs, want))
    leaves, d = ([t.detach().clone().requires_grad_() for t in sets[0][0]], sets[0][1].clone())
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        run(leaves, d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        out = run(leaves, d)
    for s, w in zip(sets, want):
        with torch.no_grad():
            for t, x in zip(leaves, s[0]):
                t.copy_(x)
            d.copy_(s[1])
        graph.replay()
        assert _same(out, w)
