"""Torch-tensor wrappers around the C ABI (one function per entry point).

These check dtypes/shapes the way the reference's wrappers assert them, pass
raw pointers and the current stream to the library and return torch tensors.
Every function requires CUDA tensors; there is no CPU path.
"""
from __future__ import annotations

import functools
import threading

import torch

from microserve_b200 import _lib
from microserve_b200._lib import check, ptr, stream_ptr

FP8 = torch.float8_e4m3fn


def _cuda(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (microserve-b200 has no CPU path)")


class _Workspace(threading.local):
    """Per-thread, per-device scratch buffers for kernels that need one, one
    buffer per kernel family ("gemm", "decode").

    The GEMM buffer starts zeroed: its first bytes hold tile flags that every
    GEMM call leaves at zero again. Buffers grow on demand outside CUDA-graph
    capture; inside a capture they must already be large enough (reserve()
    before capturing)."""

    def __init__(self):
        self.buf: dict[tuple[int, str], torch.Tensor] = {}
        # Buffers replaced by a larger one stay alive: captured CUDA graphs may
        # still hold their addresses.
        self.retired: list[torch.Tensor] = []

    def get(self, nbytes: int, device: torch.device, name: str = "decode") -> torch.Tensor | None:
        if nbytes == 0:
            return None
        idx = device.index if device.index is not None else torch.cuda.current_device()
        cur = self.buf.get((idx, name))
        if cur is None or cur.numel() < nbytes:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(
                    f"{name} workspace of {nbytes} bytes needed during CUDA-graph capture; reserve it first")
            if cur is not None:
                self.retired.append(cur)
            cur = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
            self.buf[(idx, name)] = cur
        return cur

    def reserve(self, nbytes: int, device: torch.device, name: str = "decode") -> None:
        self.get(nbytes, device, name)


workspace = _Workspace()


def quantize_rows_fp8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [M, K] fp16 (unit stride on K) -> (xq [M, K] e4m3, sx [M] fp32)."""
    _cuda(x, "x")
    if x.dtype != torch.float16:
        raise ValueError("quantize_rows_fp8 requires fp16 input")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    M, K = x2.shape
    xq = torch.empty((M, K), dtype=FP8, device=x.device)
    sx = torch.empty((M,), dtype=torch.float32, device=x.device)
    check(_lib.load().ms_quantize_rows_fp8(ptr(x2), x2.stride(0), M, K, ptr(xq), ptr(sx), stream_ptr()),
          "ms_quantize_rows_fp8")
    return xq, sx


def row_amax(x: torch.Tensor) -> torch.Tensor:
    """x [M, K] fp16 -> amax [M] fp32, the per-row absolute maximum."""
    _cuda(x, "x")
    if x.dtype != torch.float16:
        raise ValueError("row_amax requires fp16 input")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    M, K = x2.shape
    amax = torch.empty((M,), dtype=torch.float32, device=x.device)
    check(_lib.load().ms_row_amax(ptr(x2), x2.stride(0), M, K, ptr(amax), stream_ptr()), "ms_row_amax")
    return amax


def quantize_rows_fp8_amax(x: torch.Tensor, amax: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """quantize_rows_fp8 with the row amax given (scale = max(amax, 1e-8) * fl32(1/448))."""
    _cuda(x, "x")
    if x.dtype != torch.float16 or amax.dtype != torch.float32:
        raise ValueError("quantize_rows_fp8_amax requires fp16 rows and fp32 amax")
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    M, K = x2.shape
    if amax.shape != (M,):
        raise ValueError("amax must have one entry per row")
    xq = torch.empty((M, K), dtype=FP8, device=x.device)
    sx = torch.empty((M,), dtype=torch.float32, device=x.device)
    check(_lib.load().ms_quantize_rows_fp8_amax(ptr(x2), x2.stride(0), M, K, ptr(amax), ptr(xq), ptr(sx),
                                                stream_ptr()), "ms_quantize_rows_fp8_amax")
    return xq, sx


def fp8_gemm(xq: torch.Tensor, sx: torch.Tensor, wq: torch.Tensor, sw: torch.Tensor,
             bias: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """y [M, N] fp16 = fp16((xq . wq^T) * sx[:, None] * sw[None, :]) (+ bias)."""
    _cuda(xq, "xq")
    M, K = xq.shape
    N = wq.shape[0]
    if wq.shape[1] != K or xq.dtype != FP8 or wq.dtype != FP8:
        raise ValueError("fp8_gemm: expected e4m3 xq [M, K] and wq [N, K]")
    if not (xq.is_contiguous() and wq.is_contiguous()):
        raise ValueError("fp8_gemm: operands must be contiguous")
    y = out if out is not None else torch.empty((M, N), dtype=torch.float16, device=xq.device)
    lib = _lib.load()
    nbytes = lib.ms_fp8_gemm_workspace_size(M, N, K)
    ws = workspace.get(nbytes, xq.device, "gemm")
    check(lib.ms_fp8_gemm(ptr(xq), ptr(sx), ptr(wq), ptr(sw), ptr(bias), ptr(y), M, N, K, ptr(ws),
                          0 if ws is None else ws.numel(), stream_ptr()), "ms_fp8_gemm")
    return y


def f16_gemm(x: torch.Tensor, w: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """y [M, N] fp16 = x [M, K] . w [N, K]^T with fp32 accumulation (the LM head's
    F.linear) on this library's tcgen05 GEMM."""
    _cuda(x, "x")
    M, K = x.shape
    N = w.shape[0]
    if w.shape[1] != K or x.dtype != torch.float16 or w.dtype != torch.float16:
        raise ValueError("f16_gemm: expected fp16 x [M, K] and w [N, K]")
    if not (x.is_contiguous() and w.is_contiguous()):
        raise ValueError("f16_gemm: operands must be contiguous")
    y = out if out is not None else torch.empty((M, N), dtype=torch.float16, device=x.device)
    lib = _lib.load()
    ws = workspace.get(lib.ms_f16_gemm_workspace_size(M, N, K), x.device, "gemm")
    check(lib.ms_f16_gemm(ptr(x), ptr(w), ptr(y), M, N, K, ptr(ws), 0 if ws is None else ws.numel(), stream_ptr()),
          "ms_f16_gemm")
    return y


def fp8_gemm_rowpar(xq: torch.Tensor, sx: torch.Tensor, wq: torch.Tensor, sw: torch.Tensor, bases, rank: int,
                    world: int, max_rows: int) -> None:
    """Row-parallel FP8 GEMM whose output rows go to their owners' receive slots in
    the tensor-parallel buffers `bases` (ms_fp8_gemm_rowpar)."""
    _cuda(xq, "xq")
    M, K = xq.shape
    N = wq.shape[0]
    if wq.shape[1] != K or xq.dtype != FP8 or wq.dtype != FP8:
        raise ValueError("fp8_gemm_rowpar: expected e4m3 xq [M, K] and wq [N, K]")
    if not (xq.is_contiguous() and wq.is_contiguous()):
        raise ValueError("fp8_gemm_rowpar: operands must be contiguous")
    lib = _lib.load()
    ws = workspace.get(lib.ms_fp8_gemm_workspace_size(M, N, K), xq.device, "gemm")
    check(lib.ms_fp8_gemm_rowpar(ptr(xq), ptr(sx), ptr(wq), ptr(sw), M, N, K, ptr(ws), 0 if ws is None else ws.numel(),
                                 bases, rank, world, max_rows, stream_ptr()), "ms_fp8_gemm_rowpar")


def fp8_gemm_rowpar_ar_rmsnorm(xq: torch.Tensor, sx: torch.Tensor, wq: torch.Tensor, sw: torch.Tensor, bases,
                               rank: int, world: int, max_rows: int, residual: torch.Tensor, weight: torch.Tensor,
                               eps: float, want_fp16: bool) -> None:
    """Row-parallel FP8 GEMM + all-reduce + residual + RMSNorm + FP8 (or fp16) rows in one
    kernel over the tensor-parallel buffers `bases` (ms_fp8_gemm_rowpar_ar_rmsnorm)."""
    _cuda(xq, "xq")
    M, K = xq.shape
    N = wq.shape[0]
    if wq.shape[1] != K or xq.dtype != FP8 or wq.dtype != FP8:
        raise ValueError("fp8_gemm_rowpar_ar_rmsnorm: expected e4m3 xq [M, K] and wq [N, K]")
    if not (xq.is_contiguous() and wq.is_contiguous()):
        raise ValueError("fp8_gemm_rowpar_ar_rmsnorm: operands must be contiguous")
    lib = _lib.load()
    ws = workspace.get(lib.ms_fp8_gemm_workspace_size(M, N, K), xq.device, "gemm")
    check(lib.ms_fp8_gemm_rowpar_ar_rmsnorm(ptr(xq), ptr(sx), ptr(wq), ptr(sw), M, N, K, ptr(ws),
                                            0 if ws is None else ws.numel(), bases, rank, world, max_rows,
                                            ptr(residual), ptr(weight), float(eps), 1 if want_fp16 else 0,
                                            stream_ptr()), "ms_fp8_gemm_rowpar_ar_rmsnorm")


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: torch.Tensor | None = None,
            want_fp16: bool = True, want_fp8: bool = False):
    """(residual +) RMSNorm with optional fp16 and FP8 outputs.

    Returns (y | None, yq | None, sy | None, residual_out | None)."""
    _cuda(x, "x")
    H = x.shape[-1]
    x2 = x.reshape(-1, H)
    if not x2.is_contiguous():
        x2 = x2.contiguous()
    M = x2.shape[0]
    dev = x.device
    r2 = None
    rout = None
    if residual is not None:
        r2 = residual.reshape(-1, H)
        if not r2.is_contiguous():
            r2 = r2.contiguous()
        rout = torch.empty_like(x2)
    y = torch.empty_like(x2) if want_fp16 else None
    yq = torch.empty((M, H), dtype=FP8, device=dev) if want_fp8 else None
    sy = torch.empty((M,), dtype=torch.float32, device=dev) if want_fp8 else None
    check(_lib.load().ms_rmsnorm(ptr(x2), ptr(r2), ptr(weight), M, H, float(eps), ptr(rout), ptr(y), ptr(yq),
                                 ptr(sy), stream_ptr()), "ms_rmsnorm")
    return y, yq, sy, rout


def silu_mul(gu: torch.Tensor, want_fp16: bool = True, want_fp8: bool = False):
    """gu [M, 2I] -> (a [M, I] fp16 | None, aq | None, sa | None)."""
    _cuda(gu, "gu")
    g2 = gu.reshape(-1, gu.shape[-1])
    if not g2.is_contiguous():
        g2 = g2.contiguous()
    M, I2 = g2.shape
    I = I2 // 2
    out = torch.empty((M, I), dtype=torch.float16, device=gu.device) if want_fp16 else None
    aq = torch.empty((M, I), dtype=FP8, device=gu.device) if want_fp8 else None
    sa = torch.empty((M,), dtype=torch.float32, device=gu.device) if want_fp8 else None
    check(_lib.load().ms_silu_mul(ptr(g2), M, I, ptr(out), ptr(aq), ptr(sa), stream_ptr()), "ms_silu_mul")
    return out, aq, sa


def store_kv_fp8(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping) -> None:
    T, Hkv, D = key.shape
    check(_lib.load().ms_store_kv_fp8(ptr(key), ptr(value), T, Hkv, D, ptr(slot_mapping), ptr(k_cache),
                                      ptr(v_cache), ptr(k_scale), ptr(v_scale), stream_ptr()), "ms_store_kv_fp8")


def qkv_post(qkv: torch.Tensor, q_heads: int, kv_heads: int, head_dim: int, positions: torch.Tensor,
             cos_tab: torch.Tensor, sin_tab: torch.Tensor, q_norm_w: torch.Tensor | None,
             k_norm_w: torch.Tensor | None, eps: float, slots: torch.Tensor | None = None,
             caches: tuple | None = None, want_kv: bool = False):
    """Fused q/k norm + RoPE (+ FP8 KV store). Returns (q, k | None, v | None)."""
    T = qkv.shape[0]
    dev = qkv.device
    q = torch.empty((T, q_heads, head_dim), dtype=torch.float16, device=dev)
    k = torch.empty((T, kv_heads, head_dim), dtype=torch.float16, device=dev) if want_kv else None
    v = torch.empty((T, kv_heads, head_dim), dtype=torch.float16, device=dev) if want_kv else None
    kc = vc = ks = vs = None
    if caches is not None:
        kc, vc, ks, vs = caches
    check(_lib.load().ms_qkv_post(ptr(qkv), T, q_heads, kv_heads, head_dim, ptr(q_norm_w), ptr(k_norm_w),
                                  float(eps), ptr(positions), ptr(cos_tab), ptr(sin_tab),
                                  ptr(slots) if caches is not None else None, ptr(q), ptr(k), ptr(v), ptr(kc),
                                  ptr(vc), ptr(ks), ptr(vs), stream_ptr()), "ms_qkv_post")
    return q, k, v


def decode_workspace_bytes(B: int, Hq: int, Hkv: int, max_blocks: int, block_size: int) -> int:
    return _lib.load().ms_paged_decode_workspace_size(B, Hq, Hkv, max_blocks, block_size)


def paged_decode_fp8(query, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_tables,
                     softmax_scale: float, out: torch.Tensor | None = None) -> torch.Tensor:
    B, Hq, D = query.shape
    NB, BS, Hkv, D2 = k_cache.shape
    max_blocks = block_tables.shape[1]
    o = out if out is not None else torch.empty_like(query)
    lib = _lib.load()
    nbytes = lib.ms_paged_decode_workspace_size(B, Hq, Hkv, max_blocks, BS)
    ws = workspace.get(nbytes, query.device)
    check(lib.ms_paged_decode_fp8(ptr(query), ptr(k_cache), ptr(v_cache), ptr(k_scale), ptr(v_scale),
                                  ptr(cache_seqlens), ptr(block_tables), ptr(o), B, Hq, Hkv, D, BS, max_blocks,
                                  float(softmax_scale), ptr(ws), 0 if ws is None else ws.numel(), stream_ptr()),
          "ms_paged_decode_fp8")
    return o


def paged_prefill_fp8(query, k_cache, v_cache, k_scale, v_scale, block_tables, cu_q, kv_lens,
                      softmax_scale: float) -> torch.Tensor:
    T, Hq, D = query.shape
    NB, BS, Hkv, _ = k_cache.shape
    o = torch.empty_like(query)
    num_seqs = cu_q.shape[0] - 1
    check(_lib.load().ms_paged_prefill_fp8(ptr(query), ptr(k_cache), ptr(v_cache), ptr(k_scale), ptr(v_scale),
                                           ptr(block_tables), ptr(cu_q), ptr(kv_lens), ptr(o), num_seqs, T, Hq,
                                           Hkv, D, BS, block_tables.shape[1], float(softmax_scale), stream_ptr()),
          "ms_paged_prefill_fp8")
    return o


def varlen_prefill(q, k, v, cu, softmax_scale: float) -> torch.Tensor:
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    o = torch.empty_like(q)
    check(_lib.load().ms_varlen_prefill(ptr(q), ptr(k), ptr(v), ptr(cu), ptr(o), cu.shape[0] - 1, T, Hq, Hkv, D,
                                        float(softmax_scale), stream_ptr()), "ms_varlen_prefill")
    return o


def argmax_rows(x: torch.Tensor, want_max: bool = False):
    """Row-wise argmax of fp16 logits [M, V] (unit stride on V): int64 indices
    (first index of the maximum, NaN highest, torch.argmax's rule) and, if
    want_max, the fp32 maxima."""
    _cuda(x, "x")
    if x.dtype != torch.float16 or x.dim() != 2 or x.stride(1) != 1:
        raise ValueError("argmax_rows: expected fp16 [M, V] with unit stride on V")
    M, V = x.shape
    idx = torch.empty(M, dtype=torch.int64, device=x.device)
    vmax = torch.empty(M, dtype=torch.float32, device=x.device) if want_max else None
    lib = _lib.load()
    ws = workspace.get(lib.ms_argmax_workspace_size(M), x.device, "argmax")
    check(lib.ms_argmax_rows(ptr(x), M, V, x.stride(0), ptr(idx), ptr(vmax), ptr(ws),
                             0 if ws is None else ws.numel(), stream_ptr()), "ms_argmax_rows")
    return (idx, vmax) if want_max else idx


# ------------------------------------------------------------------ 4-bit KV cache
def fp4_cache_shapes(num_blocks: int, block_size: int, kv_heads: int, head_dim: int = 128):
    """Shapes (codes, scales) of one of the two halves (keys or values) of a 4-bit cache; both uint8."""
    return (num_blocks, kv_heads, block_size, head_dim // 2), (num_blocks, kv_heads, block_size, head_dim // 16)


def _on_current_device(what: str, *tensors: torch.Tensor) -> None:
    """Every tensor on the current CUDA device, whose current stream the kernel runs on."""
    dev = tensors[0].get_device()  # -1: not a CUDA tensor
    for t in tensors:
        if t.get_device() != dev:
            break
    else:
        if dev >= 0 and dev == _lib.current_device():
            return
    raise ValueError(f"{what}: every tensor must be on the current CUDA device, these are on "
                     f"{sorted({str(t.device) for t in tensors})} (use torch.cuda.device(...))")


def _fp4_cache(what: str, k_cache, v_cache, k_scale, v_scale, head_dim: int) -> tuple[int, int, int]:
    """Checks the four tensors of a 4-bit cache; (num_blocks, kv_heads, block_size)."""
    NB, Hkv, BS, half = shape = k_cache.shape
    if half * 2 != head_dim:
        raise ValueError(f"{what}: head_dim {head_dim} does not match a cache of {half} code bytes a row")
    scales = k_scale.shape
    if v_cache.shape != shape or v_scale.shape != scales or scales != (NB, Hkv, BS, half // 8):
        raise ValueError(f"{what}: cache shapes {tuple(shape)} {tuple(v_cache.shape)} {tuple(k_scale.shape)} "
                         f"{tuple(v_scale.shape)} do not belong together")
    u8 = torch.uint8
    if not (k_cache.dtype is u8 and v_cache.dtype is u8 and k_scale.dtype is u8 and v_scale.dtype is u8
            and k_cache.is_contiguous() and v_cache.is_contiguous() and k_scale.is_contiguous()
            and v_scale.is_contiguous()):
        raise ValueError(f"{what}: the 4-bit cache is contiguous uint8")
    return NB, Hkv, BS


def _vector_rows(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """(t, token stride, head stride) of t [T, heads, 128], itself where a kernel can read its rows as
    16-byte vectors, else a contiguous copy (of a tensor at an address that is not, a clone)."""
    ts, hs, one = t.stride()
    if one == 1 and ts % 8 == 0 and hs % 8 == 0 and t.data_ptr() % 16 == 0:
        return t, ts, hs
    t = t.contiguous() if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)
    return t, t.shape[1] * t.shape[2], t.shape[2]


def store_kv_fp4(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 k_scale: torch.Tensor, v_scale: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Quantise key / value [T, Hkv, 128] fp16 (any token and head stride) into the 4-bit cache at
    slot_mapping [T] int64 (negative: skipped; no slot twice). ms_store_kv_fp4."""
    T, Hkv, D = key.shape
    NB, H, BS = _fp4_cache("store_kv_fp4", k_cache, v_cache, k_scale, v_scale, D)
    if value.shape != key.shape or H != Hkv or key.dtype is not torch.float16 or value.dtype is not torch.float16:
        raise ValueError("store_kv_fp4: key and value must be fp16 [T, kv_heads, head_dim] of the cache's heads")
    if slot_mapping.dtype is not torch.int64 or slot_mapping.shape != (T,) or not slot_mapping.is_contiguous():
        raise ValueError("store_kv_fp4: slot_mapping must be contiguous int64 [T]")
    _on_current_device("store_kv_fp4", key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping)
    key, kts, khs = _vector_rows(key)
    value, vts, vhs = _vector_rows(value)
    check(_lib.load().ms_store_kv_fp4(key.data_ptr(), value.data_ptr(), kts, khs, vts, vhs, T, Hkv, D,
                                      slot_mapping.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                      k_scale.data_ptr(), v_scale.data_ptr(), NB, BS, stream_ptr()),
          "ms_store_kv_fp4")


def load_kv_fp4(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                slot_mapping: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The tokens at slot_mapping [T] int64 of the 4-bit cache as fp16 (k, v) [T, Hkv, 128], exactly
    the stored values (zeros for negative slots). ms_load_kv_fp4."""
    NB, Hkv, BS = _fp4_cache("load_kv_fp4", k_cache, v_cache, k_scale, v_scale, 128)
    if slot_mapping.dtype is not torch.int64 or slot_mapping.dim() != 1 or not slot_mapping.is_contiguous():
        raise ValueError("load_kv_fp4: slot_mapping must be contiguous int64 [T]")
    _on_current_device("load_kv_fp4", k_cache, v_cache, k_scale, v_scale, slot_mapping)
    T = slot_mapping.shape[0]
    k = torch.empty(T, Hkv, 128, dtype=torch.float16, device=k_cache.device)
    v = torch.empty_like(k)
    check(_lib.load().ms_load_kv_fp4(k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                                     NB, BS, T, Hkv, 128, slot_mapping.data_ptr(), k.data_ptr(), v.data_ptr(),
                                     stream_ptr()), "ms_load_kv_fp4")
    return k, v


def _fp4_query(what: str, query: torch.Tensor,
               out: torch.Tensor | None) -> tuple[torch.Tensor, int, torch.Tensor]:
    """(query whose heads a kernel can read in place, its token stride, the output tensor)."""
    if query.dtype is not torch.float16 or query.dim() != 3:
        raise ValueError(f"{what}: query must be fp16 [tokens, heads, head_dim]")
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
    elif out.shape != query.shape or out.dtype is not torch.float16 or not out.is_contiguous():
        raise ValueError(f"{what}: out must be contiguous fp16 of query's shape")
    elif out.data_ptr() % 16 != 0:
        raise ValueError(f"{what}: out must be 16-byte aligned")
    query, ts, hs = _vector_rows(query)
    row = query.shape[1] * query.shape[2]
    if ts < row or hs != query.shape[2]:  # overlapping or interleaved heads, or a single token
        query, ts = query.contiguous(), row
    return query, ts, out


def _int32(what: str, name: str, t: torch.Tensor, *shape: int) -> None:
    got = t.shape
    if t.dtype is torch.int32 and t.is_contiguous() and (
            got == shape or (shape[-1] < 0 and len(got) == len(shape) and got[:-1] == shape[:-1])):
        return
    raise ValueError(f"{what}: {name} must be contiguous int32 of shape "
                     f"[{', '.join('*' if s < 0 else str(s) for s in shape)}]")


# Workspace bytes by sizes (and device: its SMs), looked up once: the C call takes a third of a launch.
@functools.lru_cache(maxsize=1024)
def _decode_fp4_workspace(device: int, *sizes: int) -> int:
    return _lib.load().ms_paged_decode_fp4_workspace_size(*sizes)


@functools.lru_cache(maxsize=1024)
def _prefill_fp4_workspace(device: int, *sizes: int) -> int:
    return _lib.load().ms_paged_prefill_fp4_workspace_size(*sizes)


def paged_decode_fp4(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                     v_scale: torch.Tensor, cache_seqlens: torch.Tensor, block_tables: torch.Tensor,
                     softmax_scale: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """Decode attention of query [B, Hq, 128] fp16 (any token stride) over each sequence's first
    cache_seqlens[b] tokens of the 4-bit cache; 0 for an empty sequence. ms_paged_decode_fp4."""
    B, Hq, D = query.shape
    NB, Hkv, BS = _fp4_cache("paged_decode_fp4", k_cache, v_cache, k_scale, v_scale, D)
    _int32("paged_decode_fp4", "cache_seqlens", cache_seqlens, B)
    _int32("paged_decode_fp4", "block_tables", block_tables, B, -1)
    query, q_stride, o = _fp4_query("paged_decode_fp4", query, out)
    _on_current_device("paged_decode_fp4", query, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_tables, o)
    max_blocks = block_tables.shape[1]
    # a workspace of its own for every call: calls on two streams, or two captured graphs, never share one
    ws = k_cache.new_empty(_decode_fp4_workspace(o.get_device(), B, Hq, Hkv, max_blocks, BS))
    check(_lib.load().ms_paged_decode_fp4(query.data_ptr(), q_stride, k_cache.data_ptr(), v_cache.data_ptr(),
                                          k_scale.data_ptr(), v_scale.data_ptr(), NB, cache_seqlens.data_ptr(),
                                          block_tables.data_ptr(), o.data_ptr(), B, Hq, Hkv, D, BS, max_blocks,
                                          float(softmax_scale), ws.data_ptr(), ws.numel(), stream_ptr()),
          "ms_paged_decode_fp4")
    return o


def paged_prefill_fp4(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                      v_scale: torch.Tensor, block_tables: torch.Tensor, cu_q: torch.Tensor, kv_lens: torch.Tensor,
                      softmax_scale: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of new tokens query [T, Hq, 128] fp16 (any token stride) over prefix + themselves
    in the 4-bit cache, every sequence in one launch. Rows behind cu_q[-1] are not written (pass `out`
    to keep theirs; where it shares memory with query, the query is copied). ms_paged_prefill_fp4."""
    T, Hq, D = query.shape
    NB, Hkv, BS = _fp4_cache("paged_prefill_fp4", k_cache, v_cache, k_scale, v_scale, D)
    num_seqs = kv_lens.shape[0]
    _int32("paged_prefill_fp4", "kv_lens", kv_lens, num_seqs)
    _int32("paged_prefill_fp4", "cu_q", cu_q, num_seqs + 1)
    _int32("paged_prefill_fp4", "block_tables", block_tables, num_seqs, -1)
    query, q_stride, o = _fp4_query("paged_prefill_fp4", query, out)
    if out is not None and T > 0:  # a CTA may read rows of the query after others have written theirs of the output
        q_at, o_at, row = query.data_ptr(), o.data_ptr(), 2 * Hq * D
        if q_at < o_at + T * row and o_at < q_at + (T - 1) * 2 * q_stride + row:
            query, q_stride = query.clone(memory_format=torch.contiguous_format), Hq * D
    _on_current_device("paged_prefill_fp4", query, k_cache, v_cache, k_scale, v_scale, block_tables, cu_q, kv_lens, o)
    max_blocks = block_tables.shape[1]
    # its own for every call, as in paged_decode_fp4
    ws = k_cache.new_empty(_prefill_fp4_workspace(o.get_device(), num_seqs, T, Hq, Hkv, max_blocks, BS))
    check(_lib.load().ms_paged_prefill_fp4(query.data_ptr(), q_stride, k_cache.data_ptr(), v_cache.data_ptr(),
                                           k_scale.data_ptr(), v_scale.data_ptr(), NB, block_tables.data_ptr(),
                                           cu_q.data_ptr(), kv_lens.data_ptr(), o.data_ptr(), num_seqs, T, Hq, Hkv,
                                           D, BS, max_blocks, float(softmax_scale), ws.data_ptr(), ws.numel(),
                                           stream_ptr()),
          "ms_paged_prefill_fp4")
    return o


# ------------------------------------------------------------------ page copies
def copy_pages(cache: torch.Tensor, scale: torch.Tensor, src: torch.Tensor, dst: torch.Tensor,
               num_tokens: torch.Tensor | None = None) -> None:
    """Copy tokens [0, num_tokens[i]) (None: whole pages) of page src[i] to page dst[i] in every plane of
    a paged cache, codes and scales in one launch. ms_copy_pages.

    cache / scale: the FP8 cache [..., NB, BS, Hkv, D] e4m3 with [..., NB, BS, Hkv] fp32, or the 4-bit one
    [..., NB, Hkv, BS, 64] with [..., NB, Hkv, BS, 8] uint8; the leading dimensions (layers, K and V) are
    planes. src, dst, num_tokens: int32 [n] on the GPU. No page may be a destination twice, or both a
    source and a destination (the pairs run in any order)."""
    fp8 = cache.dtype is FP8
    if not fp8 and cache.dtype is not torch.uint8 or cache.dim() < 4:
        raise ValueError("copy_pages: expected an FP8 cache [..., pages, page_size, heads, dim] or a 4-bit one")
    lead, (NB, a, b, row) = cache.shape[:-4], cache.shape[-4:]
    if fp8:
        ok = scale.dtype is torch.float32 and scale.shape == cache.shape[:-1]
        outer, BS, row, srow = 1, a, b * row, b * 4
    else:
        ok = scale.dtype is torch.uint8 and scale.shape == (*cache.shape[:-1], row // 8)
        outer, BS, srow = a, b, row // 8
    if not ok:
        raise ValueError(f"copy_pages: scales {scale.dtype} {tuple(scale.shape)} do not belong to a cache "
                         f"{cache.dtype} {tuple(cache.shape)}")
    if not cache.is_contiguous() or not scale.is_contiguous():
        raise ValueError("copy_pages: caches must be contiguous")
    n = src.shape[0]
    _int32("copy_pages", "src", src, n)
    _int32("copy_pages", "dst", dst, n)
    if num_tokens is not None:
        _int32("copy_pages", "num_tokens", num_tokens, n)
        _on_current_device("copy_pages", cache, scale, src, dst, num_tokens)
    else:
        _on_current_device("copy_pages", cache, scale, src, dst)
    planes = 1
    for d in lead:
        planes *= d
    pages = NB * outer * BS
    check(_lib.load().ms_copy_pages(cache.data_ptr(), pages * row, row, scale.data_ptr(), pages * srow, srow, planes,
                                    outer, BS, NB, src.data_ptr(), dst.data_ptr(), ptr(num_tokens), n, stream_ptr()),
          "ms_copy_pages")
