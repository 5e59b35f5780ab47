"""The layer functions of the 4-bit KV cache, with the arguments that the FP8 ones take: strided tables, lengths and
slots, 32-bit slots, and the attention layer in each of its modes without FP8 linears."""
import pytest
import torch

from oracle import fp4_kv as F
from tests.test_fp4_gpu import DEV, SCALE, _cache, _close, _dev, _i32, _status_clean, _tables  # noqa: F401

pytestmark = pytest.mark.gpu


def _every_other(t):
    """The same values in a tensor whose last dimension has stride 2."""
    wide = torch.full((*t.shape[:-1], 2 * t.shape[-1]), -7, dtype=t.dtype, device=t.device)
    wide[..., ::2] = t
    assert t.numel() < 2 or not wide[..., ::2].is_contiguous()
    return wide[..., ::2]


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_store_and_load_take_slots_of_any_stride_and_width(dtype):
    from microserve_b200.layers.fp4_kv_cache import allocate_fp4_kvcache, load_fp4_kvcache, store_fp4_kvcache
    H, BS, T = 3, 64, 21
    codes, scales = allocate_fp4_kvcache(4, BS, H, 128, DEV, lead=(2,))
    d = [codes[0], codes[1], scales[0], scales[1]]
    c = [t.cpu() for t in d]
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(T, H, 128, generator=g).half() for _ in range(2))
    slots = torch.randperm(4 * BS, generator=g)[:T]
    slots[4] = -1
    F.store(k, v, *c, slots)
    strided = _every_other(slots.to(dtype).to(DEV))
    store_fp4_kvcache(k.to(DEV), v.to(DEV), *d, strided)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(d, c))
    for got, a, b in zip(load_fp4_kvcache(*d, strided), c[:2], c[2:]):
        s = slots.clamp_min(0)
        ref = F.decode(a[s // BS, :, s % BS], b[s // BS, :, s % BS])
        assert torch.equal(got.cpu().double(), torch.where((slots >= 0)[:, None, None], ref, 0.0))


def test_attentions_take_strided_tables_and_lengths():
    from microserve_b200.layers.fp4_attention import fp4_decode_attention, fp4_varlen_chunk_prefill_attention
    BS, lens = 64, [150, 3, 0, 200]
    bt, NB = _tables(lens, BS, 4)
    c = _cache(NB, BS, 2, 4)
    d = _dev(c)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(4, 8, 128, generator=g).half()
    tables, n = _every_other(bt.to(DEV)), _every_other(_i32(lens))
    out = torch.empty(4, 8, 128, dtype=torch.float16, device=DEV)
    got = fp4_decode_attention(q.to(DEV), *d, n, tables, SCALE, out=out)
    assert got is out
    _close(got, *F.decode_attention(q, *c, lens, bt, SCALE))
    cu = [0, 30, 33, 33, 40]
    q = torch.randn(40, 8, 128, generator=g).half()
    got = fp4_varlen_chunk_prefill_attention(q.to(DEV), *d, tables, _every_other(_i32(cu)), n, SCALE)
    _close(got, *F.prefill_attention(q, *c, bt, cu, lens, SCALE), prefill=True)


def test_the_attention_layer_s_own_forward():
    """Attention.forward (store, then attention) on the 4-bit cache: a whole prompt, a later chunk, decode steps."""
    from microserve_b200.layers.attention import Attention
    from microserve_b200.layers.fp4_kv_cache import allocate_fp4_kvcache
    from microserve_b200.utils.context import AttentionMode, Context, reset_context, set_context
    BS, H, Hq, n = 64, 2, 8, 140
    attn = Attention(Hq, 128, SCALE, H)
    codes, scales = allocate_fp4_kvcache(5, BS, H, 128, DEV, lead=(2,))
    attn.k_cache, attn.v_cache, attn.k_scale_cache, attn.v_scale_cache = codes[0], codes[1], scales[0], scales[1]
    attn.kv_cache_dtype = "fp4_e2m1"
    c = [t.cpu() for t in (codes[0], codes[1], scales[0], scales[1])]
    g = torch.Generator().manual_seed(8)
    q, k, v = (torch.randn(n, h, 128, generator=g).half() for h in (Hq, H, H))
    table = [3, 0, 4]
    bt = torch.tensor([table], dtype=torch.int32)
    at = [(0, 50, AttentionMode.PREFILL), (50, 137, AttentionMode.CHUNK_PREFILL), (137, 138, AttentionMode.DECODE),
          (138, 139, AttentionMode.DECODE), (139, 140, AttentionMode.DECODE)]
    try:
        for lo, hi, mode in at:
            slots = torch.tensor([table[p // BS] * BS + p % BS for p in range(lo, hi)])
            cu = _i32([0, hi - lo])
            set_context(Context(mode=mode, slot_mapping=slots.to(DEV), cu_seqlens_q=cu, cu_seqlens_k=cu,
                                max_seqlen_q=hi - lo, max_seqlen_k=hi, cache_seqlens=_i32([hi]),
                                block_tables=bt.to(DEV)))
            got = attn(q[lo:hi].to(DEV), k[lo:hi].to(DEV), v[lo:hi].to(DEV))
            F.store(k[lo:hi], v[lo:hi], *c, slots)
            for a, b in zip((codes[0], codes[1], scales[0], scales[1]), c):
                assert torch.equal(a.cpu(), b)
            if mode is AttentionMode.PREFILL:  # a whole prompt attends to its own fp16 keys and values
                s = torch.einsum("qhd,khd->hqk", q[:hi].double(), k[:hi].double().repeat_interleave(4, 1)) * SCALE
                p = torch.softmax(s.masked_fill(~torch.ones(hi, hi, dtype=torch.bool).tril(), float("-inf")), -1)
                vv = v[:hi].double().repeat_interleave(4, 1)
                _close(got, torch.einsum("hqk,khd->qhd", p, vv), torch.einsum("hqk,khd->qhd", p, vv.abs()), prefill=True)
            else:
                _close(got, *F.attend(q[lo:hi], *c, bt[0], hi, SCALE), prefill=mode is AttentionMode.CHUNK_PREFILL)
    finally:
        reset_context()
