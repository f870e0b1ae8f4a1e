"""Serving with a bounded cache in 4 bits: prompts of different lengths, tokens one at a time, eviction when the cache is full, and a
second turn behind what is still there.

    python examples/serve_kv4.py [--layers 4] [--batch 8] [--slots 1024] [--tokens 256]

The model around the attention is a stand-in (random weights, a few matrix products a layer); the five attention steps are those
of a real one.  Prints what the cache takes, tokens per second, and how far the last step is from attention over the same
rows in 16 bits.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from acctransformer_b200 import Kv4Cache, Kv4Workspace, flash_attention_packed  # noqa: E402


class Layer:
    """Attention with grouped heads and its cache; two caches, since eviction moves rows from one to the other."""

    def __init__(self, hidden, N, N_kv, D, B, slots, dtype):
        self.N, self.N_kv, self.D = N, N_kv, D
        self.qkv = torch.randn(hidden, (N + 2 * N_kv) * D, device="cuda").mul_(hidden ** -0.5).to(dtype)
        self.out = torch.randn(N * D, hidden, device="cuda").mul_((N * D) ** -0.5).to(dtype)
        self.cache, self.spare = (Kv4Cache(B, N_kv, slots, D, dtype=dtype) for _ in range(2))
        self.weights = torch.zeros(B, N_kv, slots, device="cuda")

    def project(self, x):      # [T, hidden] -> q [T, N, D], k, v [T, N_kv, D] (views: the operators take strides)
        return (x @ self.qkv).view(-1, self.N + 2 * self.N_kv, self.D).split([self.N, self.N_kv, self.N_kv], 1)

    def prompts(self, x, lens, cu):
        """Packed rows of new tokens behind ``lens`` rows per sequence that the cache has (None: it is empty)."""
        q, k, v = self.project(x)
        if lens is None:
            y = flash_attention_packed(q, k, v, cu)
            self.cache.append(k, v, torch.zeros_like(cu[1:]), cu)
        else:
            self.cache.append(k, v, lens, cu)
            cu_all = torch.cat([cu[:1], (lens + cu.diff()).cumsum(0).int()])
            keys, values = self.cache.read(torch.zeros_like(lens), cu_all, total=int(cu_all[-1]))
            y = flash_attention_packed(q, keys, values, cu, cu_all)
        return x + y.flatten(1) @ self.out

    def token(self, x, lens, workspace):
        """One token per sequence, which attends to itself too; the probabilities that the keys get are added up."""
        q, k, v = self.project(x)
        self.cache.append(k, v, lens)
        y = self.cache.decode(q.unsqueeze(2).contiguous(), lens + 1, weights=self.weights, workspace=workspace)
        return x + y.flatten(1) @ self.out

    def evict(self, lens, keep, recent):
        _, self.weights, lens = self.cache.evict(self.weights, lens, keep, recent, self.spare)
        self.cache, self.spare = self.spare, self.cache
        return lens


def serve(layers=4, batch=8, slots=1024, tokens=256, hidden=1024, N=16, N_kv=4, D=64, dtype=torch.bfloat16, seed=0):
    torch.manual_seed(seed)
    net = [Layer(hidden, N, N_kv, D, batch, slots, dtype) for _ in range(layers)]
    workspace = Kv4Workspace(batch, N, N_kv, slots, D, "cuda", weights=True)      # one for all layers
    norm = lambda x: torch.nn.functional.rms_norm(x, (hidden,))  # noqa: E731

    def packed(sizes, lens):
        cu = torch.tensor([0] + sizes).cumsum(0).int().cuda()
        x = torch.randn(sum(sizes), hidden, device="cuda").to(dtype)
        for layer in net:
            x = norm(layer.prompts(x, lens, cu))
        return x[cu[1:].long() - 1]

    # the first turn: every slot but a few for the longest prompt
    sizes = [max(1, (slots - 8) * (i + 1) // batch) for i in range(batch)]
    x = packed(sizes, None)
    longest, lens = max(sizes), torch.tensor(sizes, dtype=torch.int32, device="cuda")
    start, stop = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    evictions = 0
    for _ in range(tokens):
        if longest == slots:      # full (the host knows without asking: lengths follow from what it has asked for)
            new = [layer.evict(lens, slots // 2, slots // 8) for layer in net]
            lens, longest, evictions = new[0], slots // 2, evictions + 1
        for layer in net:
            x = norm(layer.token(x, lens, workspace))
        lens, longest = lens + 1, longest + 1
    stop.record()

    # the second turn, behind what is in the cache (here its lengths are read back: rows have to be allocated for them)
    room = slots - int(lens.max())
    if room < batch:
        lens = [layer.evict(lens, slots // 2, slots // 8) for layer in net][0]
        room = slots - slots // 2
    sizes = [1 + (room - 1) * i // batch for i in range(batch)]
    x = packed(sizes, lens)
    lens = lens + torch.tensor(sizes, dtype=torch.int32, device="cuda")

    # the same attention from the cache a token at a time and over its rows in 16 bits
    layer = net[-1]
    cu = torch.cat([lens.new_zeros(1), lens.cumsum(0).int()])
    keys, values = layer.cache.read(torch.zeros_like(lens), cu, total=int(cu[-1]))
    q = layer.project(x)[0]
    a = layer.cache.decode(q.unsqueeze(2).contiguous(), lens, workspace=workspace).squeeze(2)
    b = flash_attention_packed(q, keys, values, torch.arange(batch + 1, device="cuda").int(), cu)
    return {"cache_bytes": sum(layer.cache.nbytes for layer in net), "bytes_in_16_bits": layers * batch * slots * N_kv * D * 4,
            "tokens_per_s": batch * tokens / start.elapsed_time(stop) * 1e3, "evictions": evictions, "lens": lens.tolist(),
            "difference": float((a.double() - b.double()).norm() / b.double().norm()), "out": x}


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("layers", 4), ("batch", 8), ("slots", 1024), ("tokens", 256)):
        parser.add_argument(f"--{name}", type=int, default=value)
    r = serve(**vars(parser.parse_args()))
    print(f"cache {r['cache_bytes'] / 1e6:.1f} MB (16 bits: {r['bytes_in_16_bits'] / 1e6:.1f} MB), {r['tokens_per_s']:.0f} tokens/s, "
          f"{r['evictions']} evictions, lengths {r['lens']}, decode against 16 bits {r['difference']:.1e}")
