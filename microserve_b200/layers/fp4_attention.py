"""Attention over the paged 4-bit KV cache, with the interfaces of the FP8 ones
(layers/fp8_decode_attention.py, layers/fp8_chunk_prefill_attention.py)."""
import torch

from microserve_b200 import kernels


def fp4_decode_attention(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                         k_scale_cache: torch.Tensor, v_scale_cache: torch.Tensor, cache_seqlens: torch.Tensor,
                         block_tables: torch.Tensor, softmax_scale: float,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """One query token per sequence [B, Hq, D] over its first cache_seqlens[b] cached tokens."""
    return kernels.paged_decode_fp4(query, k_cache, v_cache, k_scale_cache, v_scale_cache,
                                    cache_seqlens.contiguous(), block_tables.contiguous(), softmax_scale, out=out)


def fp4_varlen_chunk_prefill_attention(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                                       k_scale_cache: torch.Tensor, v_scale_cache: torch.Tensor,
                                       block_tables: torch.Tensor, cu_seqlens_q: torch.Tensor,
                                       kv_lens: torch.Tensor, softmax_scale: float,
                                       out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of every sequence of a chunked-prefill batch: sequence s has queries
    cu_seqlens_q[s]:cu_seqlens_q[s+1] and kv_lens[s] cached tokens (this chunk's included)."""
    return kernels.paged_prefill_fp4(query, k_cache, v_cache, k_scale_cache, v_scale_cache,
                                     block_tables.contiguous(), cu_seqlens_q.contiguous(), kv_lens.contiguous(),
                                     softmax_scale, out=out)
