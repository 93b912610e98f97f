"""Device-resident paged KV cache (block size 16).

Layout per layer: K and V as [num_blocks, num_kv_heads, 16, head_dim] bf16 so
that one page of one kv head is a contiguous [16, head_dim] tile (a pair of
TMA boxes for the attention kernels). All layers live in two tensors
[L, num_blocks, Hkv, 16, D]. A token's cache slot is ``block * 16 + offset``.

Replaces the reference's host-side per-sequence KV snapshots and bucketed
decode buffers (rlx-models-core src/autoregressive.rs:538-1250,
src/gpu_kv.rs:34-590; rlx-serve src/batch.rs:159-300).
"""
from __future__ import annotations

import torch

BLOCK_SIZE = 16


class PagedKVCache:
    """``dtype`` bf16; torch.float8_e4m3fn: pages then hold saturate(x / s)
    with the per-cache ``scales`` = (s_k, s_v), halving the cache's bytes and
    the decode kernel's reads (prefill reads bf16 copies of its pages); or
    torch.int8: codes with one power-of-two scale per (block, KV head) in
    ``k_scale`` / ``v_scale`` [L, num_blocks, Hkv] fp32, which follow the values
    by themselves (``ops.kv_store_int8``)."""

    def __init__(self, num_layers: int, num_blocks: int, num_kv_heads: int, head_dim: int,
                 device: torch.device | str = "cuda", dtype: torch.dtype = torch.bfloat16,
                 scales: tuple = (1.0, 1.0)):
        if dtype not in (torch.bfloat16, torch.float8_e4m3fn, torch.int8):
            raise ValueError(f"KV cache dtype {dtype}: bf16, float8_e4m3fn or int8")
        if dtype == torch.int8 and head_dim not in (64, 128):
            raise ValueError(f"int8 KV cache: head_dim 64 or 128, not {head_dim}")
        self.dtype, self.scales = dtype, (float(scales[0]), float(scales[1]))
        self.num_layers = num_layers
        self.num_blocks = num_blocks
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        shape = (num_layers, num_blocks, num_kv_heads, BLOCK_SIZE, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self.k_scale = self.v_scale = None
        if dtype == torch.int8:
            self.k_scale = torch.zeros(shape[:3], dtype=torch.float32, device=device)
            self.v_scale = torch.zeros(shape[:3], dtype=torch.float32, device=device)

    def layer(self, i: int) -> tuple[torch.Tensor, torch.Tensor]:
        return self.k[i], self.v[i]

    def int8_layer(self, i: int) -> tuple[torch.Tensor, ...]:
        """(k, v, k_scale, v_scale) of one layer of an int8 cache."""
        return self.k[i], self.v[i], self.k_scale[i], self.v_scale[i]

    rows: list | None = None  # (k, v) of every ``store_int8`` while a list is here, to store them again

    def store_int8(self, i: int, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """``ops.kv_store_int8`` into layer ``i``; ``rows`` keeps what was stored."""
        from .. import ops
        ops.kv_store_int8(k, v, slots, *self.int8_layer(i))
        if self.rows is not None:
            self.rows.append((k, v))

    def tensors(self) -> dict[str, torch.Tensor]:
        """Everything a block consists of, by name, each [L, num_blocks, ...]."""
        named = {"k": self.k, "v": self.v, "k_scale": self.k_scale, "v_scale": self.v_scale}
        return {n: t for n, t in named.items() if t is not None}

    def copy_blocks(self, src: list[int], dst: list[int]) -> None:
        """Block ``dst[i]`` becomes a copy of ``src[i]`` in every layer."""
        from .. import ops
        t = list(self.tensors().values())
        ops.kv_copy_blocks(t, t, src, dst)

    def gather_blocks(self, blocks: list[int]) -> dict[str, torch.Tensor]:
        """The blocks, in this order, in tensors of their own [L, len(blocks), ...]."""
        from .. import ops
        src = self.tensors()
        out = {n: torch.empty((t.shape[0], len(blocks)) + t.shape[2:], dtype=t.dtype, device=t.device)
               for n, t in src.items()}
        if blocks:
            ops.kv_copy_blocks(list(src.values()), list(out.values()), blocks, range(len(blocks)))
        return out

    def scatter_blocks(self, saved: dict[str, torch.Tensor], src: list[int], blocks: list[int]) -> None:
        """Blocks ``src`` of what ``gather_blocks`` returned become ``blocks`` of this cache."""
        from .. import ops
        dst = self.tensors()
        if set(saved) != set(dst):
            raise ValueError(f"KV blocks hold {sorted(saved)}, this cache {sorted(dst)}")
        if len(src):
            ops.kv_copy_blocks([saved[n].to(t.device) for n, t in dst.items()], list(dst.values()), src, blocks)

    @staticmethod
    def bytes_per_block(num_layers: int, num_kv_heads: int, head_dim: int, dtype_bytes: int = 2,
                        scale_bytes: int = 0) -> int:
        """``scale_bytes``: of one (block, KV head)'s K and V scales each (int8: 4)."""
        return 2 * num_layers * num_kv_heads * (BLOCK_SIZE * head_dim * dtype_bytes + scale_bytes)

    @classmethod
    def blocks_for_memory(cls, mem_bytes: int, num_layers: int, num_kv_heads: int, head_dim: int) -> int:
        return max(1, mem_bytes // cls.bytes_per_block(num_layers, num_kv_heads, head_dim))
