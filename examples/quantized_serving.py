"""A serving loop over an 8-bit KV cache: prompts in chunks, then decode steps, with no block list
on the host.

    python examples/quantized_serving.py [--steps 32] [--codes int8|e4m3]

Every step runs, per batch, `build_block_tables` (pages taken on the GPU from request lengths) and,
per layer, `QuantizedCache.write` and `QuantizedCache.attend`.  The layers are random projections:
the point is the cache, so the same steps run over the bf16 pool too, and the two outputs are
compared.  Prints the cache bytes of both and the relative difference of the last step's outputs.
"""
from __future__ import annotations

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


class Pages:
    """Stand-in for the engine's page allocator: this loop takes its pages on the GPU."""

    def __init__(self, count):
        self.count, self.tables = count, {}


def run(steps=32, rows=6, layers=2, hidden=512, heads=16, kv_heads=2, codes="int8", prompt=75, seed=0):
    import torch

    import shardserve_b200 as sb

    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    dim = 128
    config = dict(num_hidden_layers=layers, num_key_value_heads=kv_heads, num_attention_heads=heads,
                  hidden_size=heads * dim)
    lens = [prompt + 13 * r for r in range(rows)]
    width = (max(lens) + steps + 15) // 16
    pages = rows * width
    dtype = torch.int8 if codes == "int8" else torch.float8_e4m3fn
    small = sb.QuantizedCache(config, 1, pages, dev, dtype, allocator=Pages)
    full = sb.Cache(config, 1, pages, dev, torch.bfloat16, allocator=Pages)
    proj = torch.randn(layers, hidden, (heads + 2 * kv_heads) * dim, device=dev, generator=g) * hidden ** -0.5
    back = torch.randn(layers, heads * dim, hidden, device=dev, generator=g) * (heads * dim) ** -0.5
    proj, back = proj.bfloat16(), back.bfloat16()

    # What the loop keeps on the GPU: lengths, tables, the free list and how much of it is used.
    cached = torch.zeros(rows, dtype=torch.int32, device=dev)
    tables = torch.full((rows, width), -1, dtype=torch.int32, device=dev)
    free = torch.randperm(pages, generator=g, device=dev).int()
    head = torch.zeros(1, dtype=torch.int32, device=dev)

    def step(new, tokens, x):
        """Appends `new` tokens per row (hidden states x, both caches) and returns both outputs."""
        m = sb.build_block_tables(cached, new, tables, free, head, tokens,
                                  out={"lens": cached, "free_head": head})
        outs = []
        for cache in (small, full):
            y = x
            for layer in range(layers):
                q, k, v = (y @ proj[layer]).view(tokens, -1, dim).split([heads, kv_heads, kv_heads], 1)
                cache.write(layer, k, v, m["slots"])
                if cache is small:
                    a = cache.attend(layer, q, m["tables"], m["seqs"], m["positions"], dim ** -0.5)
                else:
                    a = sb.ragged_attention_direct(q.contiguous(), cache.k[layer], cache.v[layer], m["tables"],
                                                   m["seqs"], m["positions"], dim ** -0.5)
                y = y + a.reshape(tokens, -1) @ back[layer]
            outs.append(y)
        return outs, m

    # Prompts in two chunks, then one token per row and step.
    for part in (0, 1):
        n = [(l + 1) // 2 if part == 0 else l // 2 for l in lens]
        x = torch.randn(sum(n), hidden, device=dev, generator=g).bfloat16()
        (a, b), m = step(torch.tensor(n, dtype=torch.int32, device=dev), sum(n), x)
    one = torch.ones(rows, dtype=torch.int32, device=dev)
    for _ in range(steps):
        x = torch.randn(rows, hidden, device=dev, generator=g).bfloat16()
        (a, b), m = step(one, rows, x)
    diff = float((a.float() - b.float()).norm() / b.float().norm())
    return dict(lens=cached.tolist(), pages_used=int(head), bytes_8bit=small.bytes, bytes_bf16=full.bytes,
                relative_difference=diff, errors=sb.kernel.device_errors(dev))


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--steps", type=int, default=32)
    p.add_argument("--codes", choices=["int8", "e4m3"], default="int8")
    args = p.parse_args()
    for key, value in run(steps=args.steps, codes=args.codes).items():
        print(f"{key}: {value}")
