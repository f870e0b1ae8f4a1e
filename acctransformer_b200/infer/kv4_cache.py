"""A key/value cache held in 4 bits, for serving: a quarter to a third of the memory of a 16-bit one, and of the bytes that a
decoding step reads.

Up to 32 neighbouring values of a token's row share a minimum and a step in the cache's 16-bit type; every value is a code of 4
bits (``include/acct_b200.h`` has the formulas).  For serving: rows, queries and weights that need a gradient are refused (call
under ``torch.no_grad()``).  The cache is storage: how many slots of a sequence are in use is the caller's to know, one
``seq_lens`` tensor for all layers:

    cache = Kv4Cache(B, N_kv, S_max, D, dtype=torch.bfloat16)              # per layer, once
    out = flash_attention_packed(q, k, v, cu_seqlens)                      # the prompts ...
    cache.append(k, v, seq_lens, cu_seqlens)                               # ... go into the cache
    cache.append(k_new, v_new, seq_lens)                                   # a decoding step: one token per sequence,
    y = cache.decode(q_new, seq_lens + 1, weights=weights)                 # which attends to itself as well
    kept, weights, seq_lens = cache.evict(weights, seq_lens, keep, recent, spare)     # when it is full

The reference has no cache; the operators have no counterpart there.
"""
from __future__ import annotations

import math

import torch

from .. import _lib

__all__ = ["Kv4Cache", "Kv4Workspace"]

ROWS = 16               # rows of a record
MAX_HEAD_DIM = 128


class Kv4Workspace:
    """Caller-owned scratch for ``Kv4Cache.decode``: partial results, and the scores where probabilities are added up.  One serves
    all layers of a step.  ``num_splits``: that of the calls; 0 has room for any, -1 for calls that leave it to the library."""

    def __init__(self, B, N, N_kv, S_max, D, device, *, weights=False, num_splits=0):
        a = _lib.Kv4CacheArgs()
        a.B, a.N_kv, a.S_max, a.D = B, N_kv, S_max, D
        self.nbytes = _lib.load().acct_kv4_decode_workspace_bytes(a, N, num_splits, 1 if weights else 0)
        if self.nbytes == 0:
            raise ValueError(f"no workspace for B={B}, N={N}, S_max={S_max}, D={D}, num_splits={num_splits}")
        self.buf = torch.empty(self.nbytes, dtype=torch.uint8, device=device)


class Kv4Cache:
    """``S_max`` slots for each of ``B`` sequences and ``N_kv`` heads of width ``D`` (a multiple of 8 up to 128).

    With ``block_table`` ([B, max_pages] int32 on the device) the slots are pages of ``page_size`` rows (a power of two, 16 or
    more) out of a pool of ``num_pages`` (default: as many as the table has entries): slot s of sequence b is row
    ``s % page_size`` of page ``block_table[b, s // page_size]``.  The table may be changed in place between calls."""

    def __init__(self, B, N_kv, S_max, D, *, dtype=torch.float16, device="cuda", page_size=None, block_table=None, num_pages=None):
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"the cache's dtype must be float16 or bfloat16, got {dtype}")
        if min(B, N_kv, S_max) < 1:
            raise ValueError(f"B, N_kv and S_max must be positive, got {B}, {N_kv}, {S_max}")
        if D < 8 or D > MAX_HEAD_DIM or D % 8:
            raise ValueError(f"head_dim must be a multiple of 8 up to {MAX_HEAD_DIM}, got {D}")
        record = _lib.load().acct_kv4_record_bytes(D)
        if block_table is None:
            if page_size is not None or num_pages is not None:
                raise ValueError("page_size and num_pages go with a block_table")
            shape, page_size = (B, N_kv, -(-S_max // ROWS), record), 0
        else:
            if not isinstance(block_table, torch.Tensor) or not block_table.is_cuda:
                raise ValueError("block_table must be a CUDA tensor (this library has no CPU path)")
            if page_size is None or page_size < ROWS or page_size & (page_size - 1):
                raise ValueError(f"page_size must be a power of two of at least {ROWS}, got {page_size}")
            if block_table.dim() != 2 or block_table.shape[0] != B or block_table.shape[1] * page_size < S_max or \
                    block_table.dtype != torch.int32 or not block_table.is_contiguous():
                raise ValueError(f"block_table must be a contiguous int32 tensor [{B}, max_pages] with pages for {S_max} slots, "
                                 f"got {block_table.dtype} {tuple(block_table.shape)}")
            device = block_table.device
            num_pages = block_table.numel() if num_pages is None else num_pages
            if num_pages < 1:
                raise ValueError("num_pages must be positive")
            shape = (num_pages, N_kv, page_size // ROWS, record)
        self.B, self.N_kv, self.S_max, self.D, self.dtype, self.page_size = B, N_kv, S_max, D, dtype, page_size
        self.block_table = block_table
        self.records = torch.empty(shape, dtype=torch.uint8, device=device)
        if not self.records.is_cuda:
            raise ValueError("the cache must be on a CUDA device (this library has no CPU path)")
        self._args = (self.records, block_table, _lib.ACCT_BF16 if dtype == torch.bfloat16 else _lib.ACCT_F16, B, N_kv, S_max, D, page_size)

    @property
    def nbytes(self):
        return self.records.numel()

    def append(self, k, v, start, cu_seqlens=None):
        """Write the rows of new tokens: k, v [T, N_kv, D] (any strides that are whole 16 bytes), sequence b's being rows
        ``cu_seqlens[b]`` .. ``cu_seqlens[b + 1]``, to its slots from ``start[b]`` on.  Without ``cu_seqlens``: one token per
        sequence.  Rows that do not fit are dropped."""
        _lib.host().kv4_append(self._args, k, v, start, cu_seqlens)

    def read(self, start, cu_seqlens=None, total=None):
        """(k, v) [total, N_kv, D] of the slots that ``append`` with the same arguments wrote, as the values they stand for (a
        prefix in the cache becomes keys for ``flash_attention_packed`` again).  ``total`` = ``cu_seqlens[-1]``, which the host has
        to know."""
        if total is None:
            if cu_seqlens is not None:
                raise ValueError("total, the number of rows, goes with cu_seqlens")
            total = self.B
        return _lib.host().kv4_read(self._args, start, cu_seqlens, total)

    def decode(self, q, seq_lens=None, *, scale=None, weights=None, num_splits=0, workspace=None, out=None):
        """y[b,n,0,:] = softmax(scale * q[b,n,0,:] K[:len_b]^T) V[:len_b] for q [B, N, 1, D], N / N_kv up to 16; zeros for a
        sequence of length 0; scale defaults to D^-1/2.

        ``weights`` (float32 [B, N_kv, S_max]): the probability of every key, summed over the query heads that share it, is added
        in place."""
        if workspace is None:
            if not isinstance(q, torch.Tensor) or not q.is_cuda or q.dim() != 4:
                raise ValueError("q must be a CUDA tensor [B, N, 1, D] (this library has no CPU path)")
            workspace = Kv4Workspace(self.B, q.shape[1], self.N_kv, self.S_max, self.D, self.records.device, weights=weights is not None,
                                     num_splits=num_splits or -1)
        return _lib.host().kv4_decode(self._args, q, seq_lens, weights, 1.0 / math.sqrt(self.D) if scale is None else scale, num_splits,
                                      workspace.buf, out)

    def evict(self, weights, seq_lens, keep, recent, out):
        """Of every sequence and head the ``recent`` last slots and, of those before them, the ones with the largest ``weights``
        (equal ones: the lowest slots), ``keep`` in all, in their order to slots 0, 1, .. of ``out``, another cache of at least
        ``keep`` slots.  Returns (kept, weights, seq_lens): the slots that stay [B, N_kv, keep] (-1 behind them), their weights
        [B, N_kv, out.S_max] (0 behind them), and the new lengths, ``min(seq_lens, keep)``."""
        if not isinstance(out, Kv4Cache):
            raise ValueError("out must be a Kv4Cache")
        return _lib.host().kv4_evict(self._args, out._args, weights, seq_lens, keep, recent)
