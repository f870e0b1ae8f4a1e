"""`out` of the serving calls of linear attention: autograd notices that it is written, and it is no memory that the call reads."""
import pytest
import torch

from tests.test_linear_attention import _decays, _ours, _rand

pytestmark = pytest.mark.gpu

N, D = 4, 64


def _packed(T=40):
    q, k, v = (_rand(T, N, D, dtype=torch.bfloat16, seed=s) for s in (1, 2, 3))
    return q, k, v, _decays(N), torch.tensor([0, T], dtype=torch.int32, device="cuda")


def _calls():
    m = _ours()
    q, k, v, g, cu = _packed()
    state = torch.zeros(1, N, D, D, device="cuda")
    one = [t[:1].unsqueeze(2) for t in (q, k, v)]
    return {"packed": ((40, N, D), lambda out: m.linear_attention_packed(q, k, v, g, cu, out=out)),
            "step": ((1, N, 1, D), lambda out: m.linear_attention_step(*one, g, state, out=out))}


@pytest.mark.parametrize("call", ["packed", "step"])
def test_saved_tensors_are_noticed(call):
    shape, run = _calls()[call]
    out, w = torch.ones(shape, device="cuda", dtype=torch.bfloat16), torch.ones(shape, device="cuda", dtype=torch.bfloat16).requires_grad_()
    y = w * out      # saves out for w's gradient
    run(out)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    with torch.inference_mode():
        run(torch.empty(shape, device="cuda", dtype=torch.bfloat16))      # (has no version)


@pytest.mark.parametrize("call", ["packed", "step"])
def test_leaves_are_refused(call):
    shape, run = _calls()[call]
    leaf = torch.ones(shape, device="cuda", dtype=torch.bfloat16).requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        run(leaf)
    assert leaf.eq(1).all()
    with torch.no_grad():
        run(leaf)
    assert not leaf.eq(1).all()


def test_starts_and_decays_are_read():
    m = _ours()
    q, k, v, g, cu = _packed()
    for like in (cu, g):
        buf = torch.zeros(q.numel() * 2 + 64, dtype=torch.uint8, device="cuda")
        mine = buf[:like.nbytes].view(like.dtype).copy_(like)
        args = [mine if like is t else t for t in (g, cu)]
        with pytest.raises(ValueError, match="share memory"):
            m.linear_attention_packed(q, k, v, *args, out=buf[:q.numel() * 2].view(torch.bfloat16).view_as(q))
        m.linear_attention_packed(q, k, v, *args, out=buf[64:].view(torch.bfloat16).view_as(q))
    one = [t[:1].unsqueeze(2) for t in (q, k, v)]
    out = torch.zeros(1, N, 1, D, dtype=torch.bfloat16, device="cuda")
    mine = out.view(-1).view(torch.float32)[:N].copy_(g)
    with pytest.raises(ValueError, match="share memory"):
        m.linear_attention_step(*one, mine, torch.zeros(1, N, D, D, device="cuda"), out=out)
