"""Per-layer physical block pools of the paged KV cache (reference ``worker/paged_kv_cache.py``).

Same contract: each layer holds (key_pool, value_pool), each [num_blocks, block_size, H_kv, D],
zero-initialised (freed blocks are not cleared; readers mask by context length, and zeros keep
every stale value finite); block 0 is the null block; slot = block * block_size + offset on the
flattened [num_blocks * block_size, H_kv, D] view.  The copies run on the CUDA kernels of
``libmi_paged.so`` (one launch moves K and V of one layer).  With head partitioning each process
holds only its KV heads.

``PagedKV4CachePool`` is the same pool in 4 bits (``include/mi_kv4.h``; no counterpart in the reference):
each layer's pools are uint8 [num_blocks, H_kv, page bytes], and the same calls quantise and dequantise.
``copy_blocks`` (both kinds) copies whole blocks in every layer, for forked sequences and compaction
(``KVCacheManager.fork`` / ``compact``).
"""

from __future__ import annotations

import math
from collections.abc import Sequence

import torch

from mini_infra_b200 import ops
from mini_infra_b200.worker.kv_cache import KVCache


class PagedKVCachePool:
    def __init__(
        self,
        num_layers: int,
        num_blocks: int,
        block_size: int,
        num_kv_heads: int,
        head_dim: int,
        dtype: torch.dtype,
        device: torch.device,
    ):
        if torch.device(device).type != "cuda":
            raise RuntimeError("PagedKVCachePool lives in GPU memory; this package has no CPU path")
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        shape = (num_blocks, block_size, num_kv_heads, head_dim)
        self.kv_pools: list[tuple[torch.Tensor, torch.Tensor]] = [
            (torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))
            for _ in range(num_layers)
        ]

    @property
    def bytes_per_block(self) -> int:
        """K+V bytes of one block across all layers."""
        key_pool = self.kv_pools[0][0]
        return 2 * len(self.kv_pools) * math.prod(key_pool.shape[1:]) * key_pool.element_size()

    @property
    def total_bytes(self) -> int:
        return self.num_blocks * self.bytes_per_block

    def gather_blocks(self, block_ids: torch.Tensor) -> tuple[tuple[torch.Tensor, torch.Tensor], ...]:
        """Per layer (key, value) history [B, H_kv, nb * bs, D] (transposed views of block copies)."""
        b, nb = block_ids.shape
        shape = (b, nb * self.block_size, self.num_kv_heads, self.head_dim)
        return tuple(
            (ops.gather_blocks(kp, block_ids).view(shape).transpose(1, 2),
             ops.gather_blocks(vp, block_ids).view(shape).transpose(1, 2))
            for kp, vp in self.kv_pools
        )

    def write_prefill(
        self,
        prefill_cache: KVCache,
        token_rows: torch.Tensor,
        token_positions: torch.Tensor,
        slot_mapping: torch.Tensor,
    ) -> None:
        """Scatter every valid token of every layer: pool slot_mapping[i] <- (token_rows[i], :, token_positions[i], :)."""
        for (kp, vp), (key, value) in zip(self.kv_pools, prefill_cache):
            ops.kv_scatter(key, value, token_rows, token_positions, slot_mapping, kp, vp)

    def store_chunks(
        self,
        prefill_cache: KVCache,
        chunk_lens: torch.Tensor,
        start_positions: torch.Tensor,
        block_tables: torch.Tensor,
    ) -> None:
        """Scatter right-aligned chunks with the slots computed on the device from the block tables."""
        for (kp, vp), (key, value) in zip(self.kv_pools, prefill_cache):
            ops.kv_store_chunks(key, value, chunk_lens, start_positions, block_tables, kp, vp)

    def copy_blocks(self, pairs: Sequence[tuple[int, int]]) -> None:
        """Copy block src to block dst in every layer's key and value pool for every (src, dst), in one launch
        on the current stream.  Destinations must be distinct allocatable blocks and not be sources."""
        pairs = [(int(s), int(d)) for s, d in pairs]
        dst = [d for _, d in pairs]
        if any(not 0 <= s < self.num_blocks or not 0 < d < self.num_blocks for s, d in pairs):
            raise ValueError(f"block ids outside the pool's {self.num_blocks} blocks, or the null block as a "
                             f"destination, in {pairs}")
        if len(set(dst)) < len(dst) or set(dst) & {s for s, _ in pairs}:
            raise ValueError(f"destinations must be distinct and not be sources: {pairs}")
        if not pairs:
            return
        pools = [p for layer in self.kv_pools for p in layer]
        host = torch.tensor(pairs, dtype=torch.long).pin_memory()
        ops.kv_copy_blocks(pools, host.to(pools[0].device, non_blocking=True))


class PagedKV4CachePool(PagedKVCachePool):
    """``PagedKVCachePool`` in 4 bits; `dtype` is the model's type, in which histories are gathered."""

    def __init__(
        self,
        num_layers: int,
        num_blocks: int,
        block_size: int,
        num_kv_heads: int,
        head_dim: int,
        dtype: torch.dtype,
        device: torch.device,
    ):
        if torch.device(device).type != "cuda":
            raise RuntimeError("PagedKV4CachePool lives in GPU memory; this package has no CPU path")
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        ops.dtype_code(dtype)
        self.dtype = dtype
        shape = (num_blocks, num_kv_heads, ops.kv4_page_bytes(block_size, head_dim))
        self.kv_pools: list[tuple[torch.Tensor, torch.Tensor]] = [
            (torch.zeros(shape, dtype=torch.uint8, device=device), torch.zeros(shape, dtype=torch.uint8, device=device))
            for _ in range(num_layers)
        ]

    def gather_blocks(self, block_ids: torch.Tensor) -> tuple[tuple[torch.Tensor, torch.Tensor], ...]:
        """Per layer (key, value) history [B, H_kv, nb * bs, D] in the model's type."""
        b, nb = block_ids.shape
        shape = (b, nb * self.block_size, self.num_kv_heads, self.head_dim)
        layers = (ops.kv4_gather_blocks(kp, vp, block_ids, self.head_dim, self.dtype) for kp, vp in self.kv_pools)
        return tuple((k.view(shape).transpose(1, 2), v.view(shape).transpose(1, 2)) for k, v in layers)

    def write_prefill(
        self,
        prefill_cache: KVCache,
        token_rows: torch.Tensor,
        token_positions: torch.Tensor,
        slot_mapping: torch.Tensor,
    ) -> None:
        for (kp, vp), (key, value) in zip(self.kv_pools, prefill_cache):
            ops.kv4_scatter(key, value, token_rows, token_positions, slot_mapping, kp, vp)

    def store_chunks(
        self,
        prefill_cache: KVCache,
        chunk_lens: torch.Tensor,
        start_positions: torch.Tensor,
        block_tables: torch.Tensor,
    ) -> None:
        for (kp, vp), (key, value) in zip(self.kv_pools, prefill_cache):
            ops.kv4_store_chunks(key, value, chunk_lens, start_positions, block_tables, kp, vp)


__all__ = ["PagedKV4CachePool", "PagedKVCachePool"]
