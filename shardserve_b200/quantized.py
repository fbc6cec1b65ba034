"""Paged KV pool held in 8 bits, with the append and the attention that use it.

A pool is two code tensors [pages, 16, kv_heads, head_dim] (int8, or float8_e4m3fn) and one
float32 scale tensor [pages, kv_heads, 2]: code c of a page and KV head stands for
`c * scales[page, head, 0]` (K) or `c * scales[page, head, 1]` (V).  Half the bytes of the bf16
pool of `shardserve_b200.cache`: a GPU holds twice the tokens.  A step takes no less time for it at
present, but for attention over long contexts: on a B200, append and attention of 64 rows of U[128, 4096] 39 us
(bf16 pool 31), of 32 rows of 16 k to 32 k 68 (67; the attention alone 55 and 64), of 56 rows beside 8 prompt
chunks of 512 151 (93).  Slots, block tables, sequence ids and positions
are those of the bf16 calls (shardserve/runtime.py:28-49); the reference has no 8-bit pool.

    cache = QuantizedCache(config, world, blocks, device)
    cache.write(layer, k, v, slots)
    out = cache.attend(layer, q, tables, seqs, positions, head_dim ** -0.5)

The functions take any strides.  `QuantizedCache` lays a page of one KV head out as one run of
memory (pages, kv_heads, 16, head_dim), so that a warp that reads one head reads whole lines.

All calls launch on torch's current stream, never synchronise and allocate only their outputs
through torch; the workspace is made per device by the first call of any of them (make one
before capturing a CUDA graph).  One workspace serves a device: calls must not overlap on two
streams.  They read nothing before the kernel before them has ended.
"""
from __future__ import annotations

from typing import Any

from . import _native
from .cache import default_allocator
from .kernel import KernelUnsupported


def kv_append_q8(k_pool_layer: Any, v_pool_layer: Any, scales: Any, k: Any, v: Any,
                 slots: Any) -> None:
    """Quantises k[i], v[i] (bf16 [tokens, kv_heads, head_dim]) into row slots[i] % 16 of page
    slots[i] // 16.  Per page, head and tensor the scale becomes max(old scale, largest new
    |value| / qmax) (qmax 127 for int8, 448 for e4m3) and the codes already there are rounded to
    the new scale; writing row 0 of a page starts it anew.  Slot -1 is skipped."""
    _native.ops().kv_append_q8(k_pool_layer, v_pool_layer, scales, k, v, slots)


def kv_read_q8(k_pool_layer: Any, v_pool_layer: Any, scales: Any, slots: Any) -> Any:
    """The rows at `slots` in bf16: (k, v), each [len(slots), kv_heads, head_dim].  For moving a
    request out of the pool (to another pool, another type, the host) and for checks."""
    return _native.ops().kv_read_q8(k_pool_layer, v_pool_layer, scales, slots)


def ragged_attention_q8(q: Any, k_pool_layer: Any, v_pool_layer: Any, scales: Any,
                        block_tables: Any, query_seq_ids: Any, positions: Any,
                        sm_scale: float) -> Any:
    """`ragged_attention_direct` over an 8-bit pool: bf16 queries [tokens, heads, head_dim], one
    sequence row and absolute position per token, decode rows and prompt chunks in one call.
    Sequence id -1 marks a padding token, whose output row is zeros."""
    return _native.ops().ragged_attention_q8(q, k_pool_layer, v_pool_layer, scales, block_tables,
                                             query_seq_ids, positions, sm_scale)


class QuantizedCache:
    """8-bit counterpart of `shardserve_b200.cache.Cache`, with the same constructor; `dtype` is
    torch.int8 (default) or torch.float8_e4m3fn."""

    def __init__(self, c, world, blocks, device, dtype=None, allocator=None, scratch_pages=8):
        import torch

        dtype = torch.int8 if dtype is None else dtype
        if torch.device(device).type != "cuda" or dtype not in (torch.int8, torch.float8_e4m3fn):
            raise KernelUnsupported("the 8-bit KV pool is an int8 or float8_e4m3fn CUDA tensor")
        if scratch_pages < 0:
            raise KernelUnsupported("scratch_pages must be >= 0")
        self.blocks = (allocator or default_allocator())(blocks)
        self.scratch_pages = int(scratch_pages)
        self.shape = (c["num_hidden_layers"], blocks + self.scratch_pages, 16,
                      c["num_key_value_heads"] // world, c["hidden_size"] // c["num_attention_heads"])
        layers, pages, rows, heads, dim = self.shape

        def pool():
            raw = torch.zeros((layers, pages, heads, rows, dim), device=device, dtype=torch.int8)
            return raw.view(dtype).transpose(2, 3)

        self.k, self.v = pool(), pool()
        self.scales = torch.zeros((layers, pages, heads, 2), device=device, dtype=torch.float32)
        self.bytes = 2 * self.k.numel() + 4 * self.scales.numel()

    def write(self, layer, k, v, slots):
        """Appends k, v [tokens, kv_heads, head_dim] at `slots` of `layer`."""
        kv_append_q8(self.k[layer], self.v[layer], self.scales[layer], k, v, slots)

    def read(self, layer, slots):
        """The rows at `slots` of `layer` in bf16: (k, v)."""
        return kv_read_q8(self.k[layer], self.v[layer], self.scales[layer], slots)

    def attend(self, layer, q, block_tables, query_seq_ids, positions, sm_scale):
        """Attention of `q` over `layer`."""
        return ragged_attention_q8(q, self.k[layer], self.v[layer], self.scales[layer],
                                   block_tables, query_seq_ids, positions, sm_scale)
