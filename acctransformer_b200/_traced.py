"""Operators under torch.jit.trace.

The tracer does not see the native path: it would put the tensors that come out of it into the graph as constants.  What it records is a
Python function, which runs again on the new operands; the native operator and its gradient run inside it."""
from __future__ import annotations

import contextlib

import torch

__all__ = ["call"]


@contextlib.contextmanager
def _untraced():
    state = torch._C._get_tracing_state()
    torch._C._set_tracing_state(None)
    try:
        yield
    finally:
        torch._C._set_tracing_state(state)


class _Traced(torch.autograd.Function):
    @staticmethod
    def forward(ctx, operator, *operands):
        # a graph of its own from the operands on, if a gradient is wanted (they share the operands' memory and versions)
        wanted = ctx.needs_input_grad[1:]
        with _untraced(), torch.set_grad_enabled(any(wanted)):
            inner = [x.detach().requires_grad_(w) if isinstance(x, torch.Tensor) else x for x, w in zip(operands, wanted)]
            out = operator(*inner)
            values = tuple(x.detach() for x in out)
        ctx.inner, ctx.out = inner, out
        if not torch.jit.is_tracing():
            return values
        # tensors that the tracer has seen begin, so that it takes none for a constant
        known = tuple(torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in values)
        with _untraced():
            for a, x in zip(known, values):
                a.copy_(x)
        return known

    @staticmethod
    def backward(ctx, *grads):
        at = [i for i, x in enumerate(ctx.inner) if isinstance(x, torch.Tensor) and x.requires_grad]
        both = [(x, g) for x, g in zip(ctx.out, grads) if x.requires_grad]
        got = torch.autograd.grad([x for x, _ in both], [ctx.inner[i] for i in at], [g for _, g in both], retain_graph=True,
                                  create_graph=torch.is_grad_enabled(), allow_unused=True)
        result = [None] * len(ctx.inner)
        for i, g in zip(at, got):
            result[i] = g
        return (None, *result)


def call(operator, *operands):
    """operator(*operands), a tuple of tensors, as a trace can record it; operands are tensors or None.  `operator` prints alike each time it is
    recorded (a trace is checked against a second one by what it prints)."""
    return _Traced.apply(operator, *operands)
