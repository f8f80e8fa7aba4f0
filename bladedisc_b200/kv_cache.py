"""A paged key / value cache in 8 bits for the layers of a decoder.

The state of a serving process in one object: the levels and scales of every layer, the block table and cached
length of every request, and the stack of free blocks.  Everything lies on the GPU and is updated there by the
operators of :mod:`bladedisc_b200.ops`; no call reads it back, so a decode step can be captured into a CUDA graph.
Steps must follow one another on one stream (or be ordered by the caller): they share the state.
"""
from typing import Optional, Tuple

import torch

from . import ops


class PagedKVCache8:
    """``requests`` rows of up to ``max_seq`` tokens over ``num_blocks`` blocks of ``block_size`` tokens.

    Memory: ``2 * layers * num_blocks * kv_heads * (block_size * head_dim + 4)`` bytes.

    ``rope``: the cosines and sines of the positions that a request can reach, where a decoder keeps them with its cache:
    a step that was captured into a graph holds their addresses as it does those of the cache."""

    def __init__(self, layers: int, requests: int, num_blocks: int, kv_heads: int, head_dim: int, max_seq: int,
                 block_size: int = 64, device="cuda"):
        if block_size not in (16, 32, 64, 128):
            raise ValueError("block_size must be 16, 32, 64 or 128")
        if head_dim not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        if min(layers, requests, num_blocks, kv_heads, max_seq) < 1:
            raise ValueError("sizes must be positive")
        self.layers, self.requests, self.num_blocks, self.block_size = layers, requests, num_blocks, block_size
        self.max_seq = max_seq
        i32 = dict(dtype=torch.int32, device=device)
        shape = (layers, num_blocks, kv_heads, block_size, head_dim)
        self.k = torch.zeros(shape, dtype=torch.int8, device=device).unbind(0)
        self.v = torch.zeros(shape, dtype=torch.int8, device=device).unbind(0)
        self.k_scale = torch.zeros(shape[:3], dtype=torch.float32, device=device).unbind(0)
        self.v_scale = torch.zeros(shape[:3], dtype=torch.float32, device=device).unbind(0)
        self.lens = torch.zeros(requests, **i32)
        self.table = torch.full((requests, -(-max_seq // block_size)), -1, **i32)
        self.free_list = torch.arange(num_blocks - 1, -1, -1, **i32)  # block 0 is handed out first
        self.free_count = torch.full((1,), num_blocks, **i32)
        self.rope: Optional[Tuple[torch.Tensor, torch.Tensor]] = None

    def extend(self, tokens: torch.Tensor, max_tokens: int) -> ops.KvPlan:
        """Room for ``tokens[r]`` new tokens of each request; see :func:`ops.kv_blocks_extend`."""
        return ops.kv_blocks_extend(tokens, self.lens, self.table, self.free_list, self.free_count, self.block_size,
                                    max_tokens)

    def trim(self, keep: torch.Tensor) -> None:
        """Keeps the first ``keep[r]`` tokens of each request: 0 ends it, fewer than cached takes drafts back.  A block
        that keeps tokens keeps its scales too, those of the drafts included; see :func:`ops.kv8_append`."""
        ops.kv_blocks_trim(keep, self.lens, self.table, self.free_list, self.free_count, self.block_size)

    def append(self, layer: int, qkv: torch.Tensor, plan: ops.KvPlan, cos: Optional[torch.Tensor] = None,
               sin: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """Stores the keys and values of the batch and returns its (rotated) queries."""
        return ops.kv8_append(qkv, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer], plan.slots,
                              plan.positions if cos is not None else None, cos, sin)

    def attend(self, layer: int, q: torch.Tensor, plan: ops.KvPlan, max_q: int, max_kv: Optional[int] = None,
               scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of the batch over what is cached, its own tokens included (append first)."""
        return ops.kv8_attention(q, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer], self.table,
                                 plan.q_start, plan.q_lens, plan.kv_lens, max_q=max_q, max_kv=max_kv, scale=scale,
                                 out=out)
