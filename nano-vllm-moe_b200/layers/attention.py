"""The attention of a decode step and the paged cache that it reads.

``PagedKVCache`` holds what the reference's engine allocates per layer and hands to its attention layers as ``k_cache`` and
``v_cache`` (nanovllm/layers/attention.py, [num_blocks, block_size, kv_heads, head_dim], slot = page * block_size + offset,
slot -1 for padding), as bfloat16 or as e4m3 codes with one scale per token and head.  ``PagedAttention`` stands between
``qkv_proj`` and ``o_proj`` of a decoder layer when every sequence has one new token: it writes the token's key and value and
attends over the sequence's pages.  ``forward_quant`` hands ``o_proj`` (W8A8-static) the e4m3 codes that it would make of the
bfloat16 result, as ``RMSNorm.forward_quant`` does for ``qkv_proj``.

Prompts are the caller's: ``PagedKVCache.write`` takes their keys and values, ``PagedKVCache.read`` gives back as bfloat16 rows
what is cached of them already.
"""
from __future__ import annotations

import torch

from .. import _lib
from .layernorm import QuantizedActivation
from .module import DirectModule


class PagedKVCache:
    """Pages for the keys and values of one layer.  ``dtype``: torch.bfloat16 or torch.float8_e4m3fn.

    In memory the tokens of a page lie one behind the other per head, [block, head, token, channel]: a block of tokens that a
    query reads is one stretch of memory.  ``k`` and ``v`` (and ``k_scale``, ``v_scale``) are views of it in the order above."""

    def __init__(self, num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int, dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if dtype not in (torch.bfloat16, torch.float8_e4m3fn):
            raise ValueError(f"a cache holds bfloat16 or float8_e4m3fn, not {dtype}")
        if min(num_blocks, block_size, num_kv_heads) < 1 or head_dim % 16 or not 16 <= head_dim <= 256:
            raise ValueError(f"bad cache shape [{num_blocks}, {block_size}, {num_kv_heads}, {head_dim}] (head_dim: a multiple of 16 from 16 to 256)")
        shape = (2, num_blocks, num_kv_heads, block_size)
        e4m3 = dtype == torch.float8_e4m3fn
        pages = torch.zeros((*shape, head_dim), dtype=torch.uint8 if e4m3 else dtype, device=device)
        self.k, self.v = pages.view(dtype).transpose(2, 3).unbind(0)
        self.k_scale, self.v_scale = torch.zeros(shape, dtype=torch.float32, device=device).transpose(2, 3).unbind(0) if e4m3 else (None, None)
        self.block_size = block_size

    def write(self, k: torch.Tensor, v: torch.Tensor, slot_mapping: torch.Tensor) -> None:
        """Rows of bfloat16 [N, kv_heads, head_dim] to their slots (int32; -1 = none)."""
        _lib.host().kv_cache_write(k, v, slot_mapping, self.k, self.v, self.k_scale, self.v_scale)

    def read(self, block_tables: torch.Tensor, cu_seqlens: torch.Tensor, rows: int) -> tuple[torch.Tensor, torch.Tensor]:
        """bfloat16 (k, v) [rows, kv_heads, head_dim]: the first tokens of the sequences, one sequence behind the other.  Both lie in one
        new piece of memory: either keeps all of it alive, and is saved with all of it (``clone`` what is to be kept alone)."""
        return _lib.host().kv_cache_read(self.k, self.v, block_tables, cu_seqlens, rows, self.k_scale, self.v_scale, None, None)


class PagedAttention(DirectModule):
    """``num_heads`` and ``num_kv_heads`` are this rank's, as the reference's ``Attention`` takes them."""

    def __init__(self, num_heads: int, head_dim: int, scale: float | None = None, num_kv_heads: int | None = None):
        super().__init__()
        self.num_heads = num_heads
        self.num_kv_heads = num_kv_heads or num_heads
        if self.num_heads % self.num_kv_heads:
            raise ValueError(f"num_heads={num_heads} must be a multiple of num_kv_heads={num_kv_heads}")
        self.head_dim = head_dim
        self.scale = scale if scale is not None else head_dim ** -0.5
        self.cache: PagedKVCache | None = None

    def _attend(self, q, k, v, slot_mapping, block_tables, context_lens, out_scale):
        cache = self.cache
        if cache is not None and cache.k.size(2) != self.num_kv_heads:
            raise ValueError(f"the cache holds {cache.k.size(2)} key heads, the layer has num_kv_heads={self.num_kv_heads}")
        if not q.is_cuda:
            raise RuntimeError("fp8lin PagedAttention requires CUDA")
        if cache is None:
            raise RuntimeError("PagedAttention has no cache: assign a PagedKVCache to its .cache first")
        host, rows, d = _lib.host(), q.shape[0], self.head_dim
        if k is not None:
            host.kv_cache_write(k.view(rows, self.num_kv_heads, d), v.view(rows, self.num_kv_heads, d), slot_mapping, cache.k, cache.v,
                                cache.k_scale, cache.v_scale)
        out = host.paged_attention(q.view(rows, self.num_heads, d), cache.k, cache.v, block_tables, context_lens, self.scale, cache.k_scale,
                                   cache.v_scale, out_scale, None)
        return out.view(rows, self.num_heads * d)

    def forward(self, q: torch.Tensor, k: torch.Tensor | None, v: torch.Tensor | None, slot_mapping: torch.Tensor | None,
                block_tables: torch.Tensor, context_lens: torch.Tensor) -> torch.Tensor:
        """q [B, heads * head_dim], k and v [B, kv_heads * head_dim] (or with the heads apart; slices of qkv_proj's output will
        do) of one token per sequence; ``context_lens`` counts the new token.  -> bfloat16 [B, heads * head_dim].
        k None: the token is in the cache already."""
        return self._attend(q, k, v, slot_mapping, block_tables, context_lens, None)

    def forward_quant(self, q: torch.Tensor, k: torch.Tensor | None, v: torch.Tensor | None, slot_mapping: torch.Tensor | None,
                      block_tables: torch.Tensor, context_lens: torch.Tensor, input_scale: torch.Tensor) -> QuantizedActivation:
        """As ``forward``, for an ``o_proj`` that takes codes made with its ``input_scale``."""
        return QuantizedActivation(self._attend(q, k, v, slot_mapping, block_tables, context_lens, input_scale), input_scale)
