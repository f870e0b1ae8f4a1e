"""torch.jit.trace of linear attention and rotary positions: a traced program computes on what it is given, not what it was traced with."""
import pytest
import torch

from tests.test_linear_attention import DTYPES, _decays, _ours, _rand

pytestmark = pytest.mark.gpu

B, N, N_kv, S, D = 2, 4, 2, 200, 64


def _inputs(dtype, seed):
    q, k, v, d = (_rand(B, h, S, D, dtype=dtype, seed=10 * seed + s) for s, h in ((1, N), (2, N_kv), (3, N_kv), (4, N)))
    return (q, k, v), d


def _grads(f, ins, d, *rest):
    leaves = [t.detach().clone().requires_grad_() for t in ins]
    y = f(*leaves, *rest)
    return (y.detach(),) + torch.autograd.grad(y, leaves, d)


def _same(traced, f, dtype, *rest):
    ins, d = _inputs(dtype, 2)
    with torch.no_grad():
        assert torch.equal(traced(*ins, *rest), f(*ins, *rest))
    assert all(torch.equal(a, b) for a, b in zip(_grads(traced, ins, d, *rest), _grads(f, ins, d, *rest)))


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("needs_grad", [False, True])
def test_function(dt, padded, needs_grad):
    m, g = _ours(), _decays(N)
    f = (lambda q, k, v, g, n: m.linear_attention(q, k, v, g, seq_lens=n)) if padded else (lambda q, k, v, g: m.linear_attention(q, k, v, g))
    rest = (g, torch.tensor([S, 31], dtype=torch.int32, device="cuda")) if padded else (g,)
    ins, _ = _inputs(DTYPES[dt], 1)
    traced = torch.jit.trace(f, tuple(t.requires_grad_(needs_grad) for t in ins) + rest, check_trace=False)
    other = (_decays(N, 3), torch.tensor([77, S - 1], dtype=torch.int32, device="cuda"))[:len(rest)]
    _same(traced, f, DTYPES[dt], *other)


@pytest.mark.parametrize("axes", [0, 1, 3])
def test_cell(axes):
    m = _ours()
    cell = m.LinearAttention(N, D, rotary=m.Rotary(D, (8, 12, 12)[:axes]) if axes else None).cuda()
    ins, _ = _inputs(torch.bfloat16, 1)
    traced = torch.jit.trace(lambda q, k, v: cell(q, k, v), ins, check_trace=False)
    _same(traced, cell, torch.bfloat16)


def test_checked_trace_of_a_model():
    """As by default: the trace is made twice and compared, operands come from weights that need a gradient."""
    m = _ours()

    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.into = torch.nn.Linear(N * D, (N + 2 * N_kv) * D)
            self.cell = m.LinearAttention(N, D, rotary=m.Rotary(D, (16, 16)))

        def forward(self, x, pos):
            q, k, v = self.into(x).unflatten(-1, (-1, D)).transpose(1, 2).split([N, N_kv, N_kv], 1)
            return self.cell(q, k, v, positions=pos)
    model = Model().cuda().bfloat16()
    x, pos = _rand(B, S, N * D, dtype=torch.bfloat16, seed=1), torch.randint(0, 99, (2, B, S), device="cuda", dtype=torch.int32)
    traced = torch.jit.trace(model, (x, pos))
    x, pos = _rand(B, S, N * D, dtype=torch.bfloat16, seed=2), torch.randint(0, 99, (2, B, S), device="cuda", dtype=torch.int32)
    got, want = traced(x, pos), model(x, pos)
    assert torch.equal(got, want)
    d = torch.randn_like(want)
    assert torch.equal(*(torch.autograd.grad(y, model.into.weight, d)[0] for y in (got, want)))


@pytest.mark.parametrize("which", ["q", "k", "both"])
def test_rotary(which):
    rotary = _ours().Rotary(D, (16, 16))
    pos = torch.randint(0, 500, (2, S), device="cuda", dtype=torch.int32)
    pick = {"q": lambda q, k, p: rotary(q, None, p)[0], "k": lambda q, k, p: rotary(None, k, p)[1], "both": lambda q, k, p: rotary(q, k, p)}[which]
    (q, k, _), _ = _inputs(torch.float16, 1)
    traced = torch.jit.trace(pick, (q, k, pos), check_trace=False)
    (q, k, _), d = _inputs(torch.float16, 2)
    leaves = [q.requires_grad_(), k.requires_grad_()]
    pos = torch.randint(0, 500, (2, S), device="cuda", dtype=torch.int32)
    got, want = traced(*leaves, pos), pick(*leaves, pos)
    for a, b, leaf in zip(*((x if which == "both" else (x,)) for x in (got, want)), leaves if which == "both" else [leaves[which == "k"]]):
        assert torch.equal(a, b)
        grads = [torch.autograd.grad(x, leaf, d[:, :leaf.shape[1]], retain_graph=True)[0] for x in (a, b)]
        assert torch.equal(*grads)


def test_traced_gradients_have_their_limits():
    """As without tracing: no second derivative of linear attention, one of rotary positions; an operand that changes is noticed."""
    m, g = _ours(), _decays(N)
    ins, d = _inputs(torch.bfloat16, 1)
    traced = torch.jit.trace(lambda q, k, v: m.linear_attention(q, k, v, g), ins, check_trace=False)
    leaves = [t.clone().requires_grad_() for t in ins]
    y = traced(*leaves)
    (dq,) = torch.autograd.grad(y, leaves[0], d, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        dq.float().sum().backward()
    y = traced(*leaves)
    with torch.no_grad():
        leaves[1].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward(d)


def test_serving_is_not_traced():
    """What moves a state, or its operands, on in place is not recorded; that is an error, not a constant."""
    m, g = _ours(), _decays(N)
    rotary = m.Rotary(D)
    rows = [_rand(8, h, D, dtype=torch.bfloat16, seed=s) for s, h in ((1, N), (2, N_kv), (3, N_kv))]
    cu = torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    state, pos = torch.zeros(1, N, D, D, device="cuda"), torch.arange(8, device="cuda")
    one = [t[:1].unsqueeze(2) for t in rows]
    for f, ins in ((lambda q, k, v: m.linear_attention_packed(q, k, v, g, cu)[0], rows), (lambda q, k, v: m.linear_attention_packed(q, k, v, g, cu, state=state)[0], rows),
                   (lambda q, k, v: m.linear_attention_step(q, k, v, g, state), one), (lambda q, k, v: rotary.apply_(q, k, pos)[0], rows)):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(f, tuple(t.clone() for t in ins), check_trace=False)
