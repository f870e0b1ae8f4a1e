"""Linear attention with a decay for each head: training over batches, prompts of different lengths, single tokens.

    S_t = exp(g) S_(t-1) + k_t v_t^T,        y_t = scale S_t^T q_t  =  scale sum over i <= t of exp(g (t - i)) (q_t . k_i) v_i

with g = ``log_decay`` of the head, at most 0.  A sequence's past is its state S, [D, D] in float32 for each query head, whatever its length:

    y, state = linear_attention_packed(q, k, v, log_decay, cu_seqlens)          # the prompts
    y = linear_attention_step(q_new, k_new, v_new, log_decay, state)            # one token per sequence; the state moves on

The reference has no counterpart.
"""
from __future__ import annotations

import functools
import math

import torch

from . import _lib, _traced

__all__ = ["LinearAttention", "linear_attention", "linear_attention_packed", "linear_attention_step", "default_log_decay"]


def _scale(q, scale):
    if scale is None:
        return 1.0 / math.sqrt(max(1, q.shape[-1])) if isinstance(q, torch.Tensor) and q.dim() > 0 else 1.0
    return scale


def linear_attention(q, k, v, log_decay, *, scale=None, seq_lens=None):
    """y [B, N, S, D] of q [B, N, S, D], k and v [B, N_kv, S, D] with N_kv dividing N, float16 or bfloat16, D a multiple of 8 up to 128;
    differentiable in q, k and v.  ``log_decay``: [N], without a gradient.  ``seq_lens`` ([B] integers): rows from there on are
    padding, which nothing reads and whose outputs and gradients are 0.  scale defaults to D^-1/2."""
    y = _lib.host().linear_apply(q, k, v, log_decay, seq_lens, _scale(q, scale))
    return _traced.call(functools.partial(_recorded, scale), q, k, v, log_decay, seq_lens)[0] if y is None else y


def _recorded(scale, q, *operands):
    return (_lib.host().linear_apply(q, *operands, _scale(q, scale)),)


def linear_attention_packed(q, k, v, log_decay, cu_seqlens, *, state=None, scale=None, out=None):
    """(y, state) of packed sequences: q [T, N, D], k and v [T, N_kv, D], and an int32 tensor [B + 1] on the device with every
    sequence's first row and the end.

    ``state`` (float32 [B, N, D, D]): the states before the first rows; it is moved on in place.  Without it they are zeros, and
    the states behind the last rows come as a new tensor.  Rows that belong to no sequence are not written.  For serving: no gradient."""
    return _lib.host().linear_packed(q, k, v, log_decay, cu_seqlens, state, _scale(q, scale), out)


def linear_attention_step(q, k, v, log_decay, state, *, scale=None, out=None):
    """y [B, N, 1, D] of one token per sequence, q [B, N, 1, D], k and v [B, N_kv, 1, D], after it has gone into ``state`` (float32
    [B, N, D, D], moved on in place).  For serving: no gradient."""
    return _lib.host().linear_step(q, k, v, log_decay, state, _scale(q, scale), out)


def default_log_decay(head_num):
    """-2^(-8 (h + 1) / head_num) for head h: memories from about two tokens to some hundreds (the slopes that alibi uses)."""
    return -torch.exp2(torch.arange(1, head_num + 1, dtype=torch.float64) * (-8.0 / head_num)).float()


class LinearAttention(torch.nn.Module):
    """The cell: rotary positions, where it has a plan for them (``rotary``, a ``Rotary``), then linear attention.

    ``forward(q, k, v)`` trains on [B, N, S, D]; positions are 0, 1, .. unless given.  ``prompt`` and ``step`` serve: packed prompts
    with their states, and one token per sequence."""

    def __init__(self, head_num, head_dim, log_decay=None, scale=None, rotary=None):
        super().__init__()
        log_decay = default_log_decay(head_num) if log_decay is None else torch.as_tensor(log_decay, dtype=torch.float32)
        if tuple(log_decay.shape) != (head_num,):
            raise ValueError(f"log_decay must hold a number for each of {head_num} heads, got {tuple(log_decay.shape)}")
        if not log_decay.is_meta and (bool((log_decay > 0).any()) or bool(log_decay.isnan().any())):
            raise ValueError("log_decay must be at most 0")
        if rotary is not None and rotary.head_dim != head_dim:
            raise ValueError(f"rotary is a plan for head_dim {rotary.head_dim}, not {head_dim}")
        self.head_num, self.head_dim, self.scale, self.rotary = head_num, head_dim, scale, rotary
        self.register_buffer("log_decay", log_decay.detach().clone())

    def _apply(self, fn, recurse=True):
        decays = self.log_decay
        super()._apply(fn, recurse)
        if self.log_decay.dtype != torch.float32:      # they stay float32, whatever type the module is cast to
            device = self.log_decay.device
            self.log_decay = torch.empty_like(decays, dtype=torch.float32, device=device) if decays.is_meta else decays.to(device, torch.float32)
        return self

    def forward(self, q, k, v, seq_lens=None, positions=None):
        if self.rotary is not None:
            if positions is None:
                positions = torch.arange(q.shape[2], dtype=torch.int32, device=q.device).expand(len(self.rotary.sections), -1)
            q, k = self.rotary(q, k, positions)
        elif positions is not None:
            raise ValueError("positions go with a rotary plan")
        return linear_attention(q, k, v, self.log_decay, scale=self.scale, seq_lens=seq_lens)

    def prompt(self, q, k, v, cu_seqlens, state=None, positions=None):
        """(y, state) of packed prompts; with a rotary plan, ``positions`` of all rows."""
        q, k = self._turned(q, k, positions)
        return linear_attention_packed(q, k, v, self.log_decay, cu_seqlens, state=state, scale=self.scale)

    def step(self, q, k, v, state, positions=None):
        """y of one token per sequence; with a rotary plan, ``positions`` [axes, B, 1] (one axis: [B, 1])."""
        q, k = self._turned(q, k, positions)
        return linear_attention_step(q, k, v, self.log_decay, state, scale=self.scale)

    def _turned(self, q, k, positions):
        if (self.rotary is None) != (positions is None):
            raise ValueError("positions and a rotary plan go together")
        return (q, k) if positions is None else self.rotary(q, k, positions)
