"""Drop-in store_kvcache for nanovllm/layers/attention.py, and the calls of a
layer whose paged cache is held in 8 bits.

The reference writes each new token's K and V rows into the paged cache with
a Triton kernel launched once per layer per step (attention.py:10-40). This
module keeps its signature and layout assertions and runs libkvoff's
16-byte-vectorized scatter instead: one launch, 64-bit slot offsets, slots of
-1 skipped, no allocation or host synchronization (CUDA-graph capturable).
"""

from __future__ import annotations

import torch

from kvoff import ops


def store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                  v_cache: torch.Tensor, slot_mapping: torch.Tensor):
    ops.store_kvcache(key, value, k_cache, v_cache, slot_mapping)


def rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, **options):
    """Rotary positions of q and k, in place by default; see kvoff.ops.rotary."""
    return ops.rotary(q, k, positions, table, **options)


def store_kvcache_fp8(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                      v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                      slot_mapping: torch.Tensor):
    """store_kvcache for an e4m3 cache with block scales; see kvoff.ops.store_kvcache_fp8."""
    ops.store_kvcache_fp8(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping)


def attention_fp8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  k_scale: torch.Tensor, v_scale: torch.Tensor, block_tables: torch.Tensor,
                  context_lens: torch.Tensor, **options) -> torch.Tensor:
    """Attention over an e4m3 paged cache; see kvoff.ops.attention_fp8."""
    return ops.attention_fp8(q, k_cache, v_cache, k_scale, v_scale, block_tables, context_lens,
                             **options)
