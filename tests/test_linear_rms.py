"""Linear attention's outputs against the definition in 64 bits, by the root mean square of each head's errors.

The bound of test_linear_attention.py adds up every term's largest error; over a slow decay's thousands of terms that is far more than their
sum, which grows like the root of their number.  Here, with every rounding an independent error of rms u / sqrt(3) of the value or less
(u = eps / 2; uniform over a step of at most 2 u |x|):

* the output is rounded once: u / sqrt(3) rms(y);
* of P C every term (a_r . b_i) l^(r-i) c_i has an error of its own, whose squares add up: over a head rms(P C terms' root of squares), of
  A S the rounding of S: the same with the state's elements as terms.  For random a, b, c with zero mean the root of the sum of squares of either
  part is rms(y) itself, so together at most u / sqrt(3) rms(y) sqrt(2).

Together u rms(y) at most; 2 u rms(y) leaves a factor of two for what random operands do not satisfy exactly."""
import pytest
import torch

from tests.test_linear_attention import DTYPES, _heads, _ours, _rand, attend

pytestmark = pytest.mark.gpu

DECAYS = [0.0, -1e-4, -0.002, -0.01, -0.07, -0.3, -2.0, -120.0]


def _check(got, want, dtype):
    u = torch.finfo(dtype).eps / 2
    for h in range(want.shape[0]):
        off = (got[h].double() - want[h]).square().mean().sqrt() / want[h].square().mean().sqrt() / u
        assert off <= 2, f"head {h} of decay {DECAYS[h % len(DECAYS)]}: {off:.2f} u"


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("N_kv,S,D", [(8, 2500, 128), (2, 1000, 64), (8, 6000, 64), (4, 640, 80)])
def test_outputs_and_gradients(dt, N_kv, S, D):
    m, N, dtype = _ours(), 8, DTYPES[dt]
    g = torch.tensor(DECAYS, device="cuda")
    q, dy = (_rand(1, N, S, D, dtype=dtype, seed=s).requires_grad_() for s in (1, 2))
    k, v = (_rand(1, N_kv, S, D, dtype=dtype, seed=s).requires_grad_() for s in (3, 4))
    y = m.linear_attention(q, k, v, g)
    dq, dk, dv = torch.autograd.grad(y, (q, k, v), dy.detach())
    xq, xd = q[0].detach().double(), dy[0].detach().double()
    xk, xv = (_heads(t[0].detach().double(), N) for t in (k, v))
    scale = D ** -0.5
    back = lambda *ops: attend(*(t.flip(1) for t in ops), g)[0].flip(1)  # noqa: E731
    shared = lambda t: t.unflatten(0, (N_kv, -1)).sum(1)  # noqa: E731
    for got, want in ((y, attend(xq, xk, xv, g)[0]), (dq, attend(xd, xv, xk, g)[0]), (dk, shared(back(xv, xd, xq))), (dv, shared(back(xk, xq, xd)))):
        _check(got[0], want * scale, dtype)


@pytest.mark.parametrize("dt", sorted(DTYPES))
@pytest.mark.parametrize("D", [64, 128])
def test_prompts_with_states(dt, D):
    m, N, dtype, n = _ours(), 8, DTYPES[dt], 1500
    g = torch.tensor(DECAYS, device="cuda")
    q, k, v = (_rand(n, N, D, dtype=dtype, seed=s) for s in (1, 2, 3))
    state = _rand(1, N, D, D, dtype=torch.float32, seed=4, scale=10.0)
    want, _ = attend(*(t.transpose(0, 1).double() for t in (q, k, v)), g, state[0])
    y, _ = m.linear_attention_packed(q, k, v, g, torch.tensor([0, n], dtype=torch.int32, device="cuda"), state=state)
    _check(y.transpose(0, 1), want * D ** -0.5, dtype)
