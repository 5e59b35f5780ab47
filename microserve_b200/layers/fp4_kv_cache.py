"""Paged 4-bit KV cache (e2m1 codes, one 8-bit scale per 16 elements): its layout,
writer and reader. No counterpart in the reference, whose cache is FP8 or fp16."""
import torch

from microserve_b200 import kernels


def allocate_fp4_kvcache(num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int, device,
                         lead: tuple[int, ...] = ()) -> tuple[torch.Tensor, torch.Tensor]:
    """Zeroed codes [*lead, num_blocks, num_kv_heads, block_size, head_dim / 2] and scales
    [*lead, num_blocks, num_kv_heads, block_size, head_dim / 16], uint8 (zeros stand for zeros)."""
    codes, scales = kernels.fp4_cache_shapes(num_blocks, block_size, num_kv_heads, head_dim)
    return (torch.zeros(*lead, *codes, dtype=torch.uint8, device=device),
            torch.zeros(*lead, *scales, dtype=torch.uint8, device=device))


def store_fp4_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      k_scale_cache: torch.Tensor, v_scale_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """store_fp8_kvcache for the 4-bit cache."""
    slot_mapping = slot_mapping.contiguous()
    if slot_mapping.dtype != torch.int64:
        slot_mapping = slot_mapping.long()
    kernels.store_kv_fp4(key, value, k_cache, v_cache, k_scale_cache, v_scale_cache, slot_mapping)


def load_fp4_kvcache(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale_cache: torch.Tensor,
                     v_scale_cache: torch.Tensor, slot_mapping: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The stored tokens at slot_mapping as fp16 key, value [T, num_kv_heads, head_dim]."""
    slot_mapping = slot_mapping.contiguous()
    if slot_mapping.dtype != torch.int64:
        slot_mapping = slot_mapping.long()
    return kernels.load_kv_fp4(k_cache, v_cache, k_scale_cache, v_scale_cache, slot_mapping)
