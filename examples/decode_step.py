"""A decoder layer served from a paged key-value cache: prompts in, then one token per sequence a step.

    python examples/decode_step.py [--steps 64] [--budget 96]

The layer is an FP8 MHA cell over a bf16 cache and a SwiGLU block of 4-bit layers with group scales.
Prompts of different lengths go through `mha_prefill`; a step then runs `mha_decode` (projections,
append, attention with its weights summed), the block, and `evict`, which keeps every sequence within
its budget of slots. The step is captured in a CUDA graph once and replayed: the lengths live on the
device. Weights and inputs are random; what is printed is the time of a step and the cache's state.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.abspath(os.path.join(os.path.dirname(__file__), "..")))

import welvet.cuda_b200 as W  # noqa: E402
from welvet.cuda_b200 import decode as D  # noqa: E402


class Pages:
    """The host's side of a cache: which pages are free, and the table row of each sequence."""

    def __init__(self, pages: int, sequences: int, per_sequence: int):
        self.free = list(range(pages))
        self.rows = [[] for _ in range(sequences)]
        self.table = torch.zeros((sequences, per_sequence), dtype=torch.int32, device="cuda")

    def reserve(self, sequence: int, slots: int, page: int) -> None:
        """Pages for `slots` slots of a sequence (those it has stay)."""
        row = self.rows[sequence]
        while len(row) * page < slots:
            row.append(self.free.pop())
        self.table[sequence, : len(row)] = torch.tensor(row, dtype=torch.int32)


def norm(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)


class Layer:
    """h = x + attention(norm(x)), then h + down(silu(gate(norm(h))) * up(norm(h)))."""

    def __init__(self, d_model: int, heads: int, kv_heads: int, inter: int, prompts, budget: int, slack: int, page: int = 16,
                 max_seq_len: int = 512, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        dim, n = d_model // heads, len(prompts)

        def weight(out, in_):
            return torch.randn((out, in_), generator=g, device="cuda") * in_ ** -0.5

        self.cell = W.MhaCell(weight(d_model, d_model), weight(kv_heads * dim, d_model), weight(kv_heads * dim, d_model),
                              weight(d_model, d_model), d_model, heads, kv_heads, max_seq_len=max_seq_len, dtype=W.FP8E4M3)
        self.gate = D.GroupDense.quantize(weight(inter, d_model), 64, D.INT4, act=W.SILU)
        self.up = D.GroupDense.quantize(weight(inter, d_model), 64, D.INT4)
        self.down = D.GroupDense.quantize(weight(d_model, inter), 64, D.UINT4)
        self.budget, self.slack = budget, slack
        slots = max(max(prompts), budget + slack) + 1
        per = -(-slots // page)
        self.pages = Pages(n * per, n, per)
        for s in range(n):
            self.pages.reserve(s, slots, page)
        shape = (n * per, page, kv_heads, dim)
        records = (n, kv_heads, per * page)
        self.cache = D.PagedKV(torch.zeros(shape, dtype=torch.bfloat16, device="cuda"),
                               torch.zeros(shape, dtype=torch.bfloat16, device="cuda"), self.pages.table,
                               torch.zeros(n, dtype=torch.int32, device="cuda"), num_heads=heads,
                               seen=torch.zeros(n, dtype=torch.int32, device="cuda"),
                               weights=torch.zeros(records, device="cuda"),
                               positions=torch.zeros(records, dtype=torch.int32, device="cuda"))
        self.att = torch.empty((n, d_model), device="cuda")
        self.h = [torch.empty((n, inter), device="cuda") for _ in range(2)]
        self.out = torch.empty((n, d_model), device="cuda")

    def prompt(self, sequence: int, x):
        y = torch.empty_like(x)
        D.mha_prefill(self.cell, self.cache, sequence, norm(x), y)
        return x + y

    def step(self, x, evict: bool = True):
        """One token per sequence: x [sequences, d_model] -> self.out."""
        D.mha_decode(self.cell, self.cache, norm(x), self.att, accumulate=True)
        self.att.add_(x)
        z = norm(self.att)
        self.gate.forward(z, self.h[0])
        self.up.forward(z, self.h[1])
        self.h[0].mul_(self.h[1])
        self.down.forward(self.h[0], self.out)
        self.out.add_(self.att)
        if evict:
            self.cache.evict(self.budget, budget=self.budget + self.slack, sinks=2, recent=self.budget // 4)
        return self.out


def run(steps: int = 64, budget: int = 96, d_model: int = 1024, heads: int = 8, kv_heads: int = 2, inter: int = 2816,
        prompts=(64, 7, 90, 33), seed: int = 0, quiet: bool = False):
    """(layer, outputs of each step) after `steps` replays of the captured step."""
    layer = Layer(d_model, heads, kv_heads, inter, prompts, budget, slack=8, seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    for s, n in enumerate(prompts):
        layer.prompt(s, torch.randn((n, d_model), generator=g, device="cuda"))
    x = torch.randn((len(prompts), d_model), generator=g, device="cuda")
    layer.step(x)  # allocates the cell's work buffers
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.step(x)
    outs = []
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize()
    start.record()
    for _ in range(steps):
        graph.replay()
        outs.append(layer.out.clone())
        x.copy_(layer.out)
    end.record()
    torch.cuda.synchronize()
    layer.cache.check_error()
    if not quiet:
        print(f"{len(prompts)} sequences, {steps} steps: {start.elapsed_time(end) / steps * 1e3:.1f} us a step; "
              f"slots in use {layer.cache.lens.tolist()}, tokens seen {layer.cache.seen.tolist()}")
    return layer, outs


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--budget", type=int, default=96)
    a = ap.parse_args()
    run(a.steps, a.budget)
