"""The 4-bit KV cache and page copies without a GPU: argument checks at the C ABI and in
the wrappers, fake ops, the fork of a sequence in the block manager and the scheduler."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import microserve_b200.library  # noqa: F401  (registers the ops)
from microserve_b200 import _lib, kernels
from microserve_b200.engine.block_manager import BlockManager
from microserve_b200.engine.scheduler import Scheduler
from microserve_b200.engine.sequence import Sequence, SequenceStatus
from oracle import fp4_kv as F

P = 1 << 20  # a 16-byte aligned address that is never read (every call below is refused before a launch)


def _store(T=4, heads=8, dim=128, k=P, slots=P, cache=P, scale=P, blocks=4, bs=256, ts=1024, hs=128):
    return _lib.load().ms_store_kv_fp4(k, P, ts, hs, 1024, 128, T, heads, dim, slots, cache, P, scale, P, blocks, bs,
                                       None)


def _decode(q=P, qs=2048, cache=P, blocks=4, lens=P, tables=P, B=2, Hq=16, Hkv=8, dim=128, bs=256, mb=4,
            ws=P, wb=1 << 30, scale=0.1):
    return _lib.load().ms_paged_decode_fp4(q, qs, cache, P, P, P, blocks, lens, tables, P, B, Hq, Hkv, dim, bs, mb,
                                           scale, ws, wb, None)


def _prefill(q=P, qs=2048, cache=P, blocks=4, tables=P, cu=P, n=2, T=9, Hq=16, Hkv=8, dim=128, bs=256, mb=4,
             scale=0.1, ws=P, wb=1 << 40):
    return _lib.load().ms_paged_prefill_fp4(q, qs, cache, P, P, P, blocks, tables, cu, P, P, n, T, Hq, Hkv, dim, bs,
                                            mb, scale, ws, wb, None)


def _copy(cache=P, cs=1 << 30, row=1024, scale=P, ss=1 << 30, srow=32, planes=2, outer=1, bs=256, pages=8, src=P,
          n=1):
    return _lib.load().ms_copy_pages(cache, cs, row, scale, ss, srow, planes, outer, bs, pages, src, P, None, n, None)


INVALID, UNSUPPORTED = _lib.MS_ERR_INVALID, _lib.MS_ERR_UNSUPPORTED


@pytest.mark.parametrize("fn,kw,rc", [
    (_store, dict(T=0), 0), (_store, dict(T=-1), INVALID), (_store, dict(dim=64), UNSUPPORTED),
    (_store, dict(bs=96), UNSUPPORTED), (_store, dict(bs=0), INVALID), (_store, dict(blocks=0), INVALID),
    (_store, dict(blocks=1 << 24), UNSUPPORTED), (_store, dict(k=None), INVALID), (_store, dict(k=P + 8), INVALID),
    (_store, dict(ts=1020), INVALID), (_store, dict(hs=4), INVALID), (_store, dict(slots=None), INVALID),
    (_store, dict(cache=None), INVALID), (_store, dict(scale=P + 4), INVALID), (_store, dict(heads=0), INVALID),
    (_decode, dict(B=0), 0), (_decode, dict(B=-1), INVALID), (_decode, dict(Hq=12), UNSUPPORTED),
    (_decode, dict(Hq=72), UNSUPPORTED), (_decode, dict(dim=96), UNSUPPORTED), (_decode, dict(bs=32), UNSUPPORTED),
    (_decode, dict(q=P + 2), INVALID), (_decode, dict(qs=2000), INVALID), (_decode, dict(qs=1024), INVALID),
    (_decode, dict(lens=None), INVALID), (_decode, dict(tables=None), INVALID), (_decode, dict(mb=0), INVALID),
    (_decode, dict(ws=None), _lib.MS_ERR_WORKSPACE), (_decode, dict(wb=100), _lib.MS_ERR_WORKSPACE),
    (_decode, dict(ws=P + 8), INVALID), (_decode, dict(scale=0.0), INVALID), (_decode, dict(scale=-1.0), INVALID),
    (_decode, dict(scale=float("nan")), INVALID), (_prefill, dict(scale=float("inf")), INVALID),
    (_prefill, dict(ws=None), _lib.MS_ERR_WORKSPACE), (_prefill, dict(wb=64), _lib.MS_ERR_WORKSPACE),
    (_prefill, dict(ws=P + 8), INVALID),
    (_prefill, dict(n=0), 0), (_prefill, dict(T=0), 0), (_prefill, dict(T=1 << 31), INVALID),
    (_prefill, dict(Hq=9), UNSUPPORTED), (_prefill, dict(cu=None), INVALID), (_prefill, dict(q=None), INVALID),
    (_prefill, dict(bs=100), UNSUPPORTED), (_prefill, dict(Hkv=0), INVALID),
    (_copy, dict(n=0), 0), (_copy, dict(planes=0), 0), (_copy, dict(n=-1), INVALID), (_copy, dict(row=6), UNSUPPORTED),
    (_copy, dict(srow=2), UNSUPPORTED), (_copy, dict(cs=1 << 10), INVALID), (_copy, dict(cs=(1 << 30) + 8), INVALID),
    (_copy, dict(cache=P + 4), INVALID), (_copy, dict(src=None), INVALID), (_copy, dict(pages=0), INVALID),
    (_copy, dict(outer=0), INVALID),
])
def test_c_abi_refuses_without_a_launch(fn, kw, rc):
    n0 = _lib.load().ms_launch_count()
    assert fn(**kw) == rc
    assert rc == 0 or _lib.load().ms_last_error()
    assert _lib.load().ms_launch_count() == n0


def _cpu_cache(NB=3, BS=64, H=2):
    codes, scales = kernels.fp4_cache_shapes(NB, BS, H)
    z = lambda s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    return z(codes), z(codes), z(scales), z(scales)


def test_wrappers_refuse_before_the_library():
    c = _cpu_cache()
    x, slots = torch.zeros(4, 2, 128, dtype=torch.float16), torch.zeros(4, dtype=torch.int64)
    lens, bt = torch.ones(4, dtype=torch.int32), torch.zeros(4, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="current CUDA device"):
        kernels.store_kv_fp4(x, x, *c, slots)
    with pytest.raises(ValueError, match="fp16"):
        kernels.store_kv_fp4(x.float(), x.float(), *c, slots)
    with pytest.raises(ValueError, match="fp16"):
        kernels.store_kv_fp4(x[:, :1], x[:, :1], *c, slots)
    with pytest.raises(ValueError, match="int64"):
        kernels.store_kv_fp4(x, x, *c, slots.int())
    with pytest.raises(ValueError, match="int64"):
        kernels.store_kv_fp4(x, x, *c, slots[:3])
    with pytest.raises(ValueError, match="head_dim"):
        kernels.store_kv_fp4(x[..., :64], x[..., :64], *c, slots)
    with pytest.raises(ValueError, match="uint8"):
        kernels.load_kv_fp4(c[0].char(), c[1].char(), c[2], c[3], slots)
    with pytest.raises(ValueError, match="belong together"):
        kernels.load_kv_fp4(c[0], c[1], c[2][:2], c[3], slots)
    with pytest.raises(ValueError, match="cache_seqlens"):
        kernels.paged_decode_fp4(x, *c, lens.long(), bt, 0.1)
    with pytest.raises(ValueError, match="block_tables"):
        kernels.paged_decode_fp4(x, *c, lens, bt[:3], 0.1)
    with pytest.raises(ValueError, match="out must be"):
        kernels.paged_decode_fp4(x, *c, lens, bt, 0.1, out=x.float())
    with pytest.raises(ValueError, match="cu_q"):
        kernels.paged_prefill_fp4(x, *c, bt, lens, lens, 0.1)
    with pytest.raises(ValueError, match="current CUDA device"):
        kernels.paged_prefill_fp4(x, *c, bt, torch.zeros(5, dtype=torch.int32), lens, 0.1)
    page = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="do not belong"):
        kernels.copy_pages(c[0], c[2].float(), page, page)
    with pytest.raises(ValueError, match="expected an FP8 cache"):
        kernels.copy_pages(c[0].float(), c[2], page, page)
    with pytest.raises(ValueError, match="dst"):
        kernels.copy_pages(c[0], c[2], page, page.long())
    with pytest.raises(ValueError, match="current CUDA device"):
        kernels.copy_pages(c[0], c[2], page, page)


def test_fake_outputs():
    ops = torch.ops.microserve_b200
    with FakeTensorMode():
        e = lambda *s, dtype=torch.float16: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
        codes, scales = kernels.fp4_cache_shapes(6, 256, 8)
        c = (e(*codes, dtype=torch.uint8), e(*codes, dtype=torch.uint8), e(*scales, dtype=torch.uint8),
             e(*scales, dtype=torch.uint8))
        slots, i32 = e(5, dtype=torch.int64), torch.int32
        assert ops.store_kv_fp4(e(5, 8, 128), e(5, 8, 128), *c, slots) is None
        k, v = ops.load_kv_fp4(*c, slots)
        assert k.shape == v.shape == (5, 8, 128) and k.dtype == torch.float16
        o = ops.paged_decode_fp4(e(4, 32, 128), *c, e(4, dtype=i32), e(4, 3, dtype=i32), 0.1)
        assert o.shape == (4, 32, 128)
        o = ops.paged_prefill_fp4(e(9, 32, 128), *c, e(2, 3, dtype=i32), e(3, dtype=i32), e(2, dtype=i32), 0.1)
        assert o.shape == (9, 32, 128)
        assert ops.copy_pages(c[0], c[2], e(2, dtype=i32), e(2, dtype=i32), None) is None


def test_oracle_rounding_points():
    """The format's definition at its corners: ties, saturation, tiny and non-finite groups."""
    x = torch.zeros(9, 128, dtype=torch.float16)
    x[0, :9] = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25])  # scale 1: every tie
    x[1, 0], x[1, 1] = 65504, float("inf")
    x[2, 0], x[2, 1] = float("nan"), 3.0
    x[3, 0] = -0.0
    x[4, 0] = 2.0 ** -24  # far below the smallest scale: stored as zero
    x[5, 16] = 6 * 2.0 ** -17  # the smallest scale, in the second group
    x[6, 0] = 6.5  # scale rn(1.0833) = 1.125
    x[7, 0] = 6 * 1.0625  # a / 6 on a scale tie (1.0625): to the even code, 1.0
    x[8, 0] = 6 * 1.1875  # tie between 1.125 and 1.25: to 1.25
    c, s = F.encode(x)
    v = F.decode(c, s)
    assert s[0, 0] == 15 * 8 and v[0, :9].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, -0.0]
    assert s[1, 0] == 226 and v[1, 0] == v[1, 1] == 61440
    assert s[2, 0] == 255 and v[2, :16].isnan().all() and (v[2, 16:] == 0).all()
    assert (v[3] == 0).all() and c[3, 0] == 8 and (v[4] == 0).all()
    assert s[5, 1] == 1 and v[5, 16] == 6 * 2.0 ** -17
    assert F.scale_value(s[6, 0]) == 1.125 and F.scale_value(s[7, 0]) == 1.0 and F.scale_value(s[8, 0]) == 1.25


# ------------------------------------------------------------------ forks
def _running(sched, n, max_tokens=64):
    seq = Sequence(list(range(n)), max_tokens=max_tokens)
    sched.add(seq)
    batch = sched.schedule()
    sched.postprocess(batch, [7] * len(batch))
    return seq


def _fork(sched, seq):
    child = Sequence(seq.token_ids, max_tokens=seq.max_tokens)
    child.num_prompt_tokens = seq.num_prompt_tokens
    return child, sched.fork(seq, child)


def test_fork_shares_full_blocks_and_copies_the_last():
    sched = Scheduler(8, 4, max_num_seqs=4)
    seq = _running(sched, 10)  # blocks 0, 1 full, 2 holds two tokens
    child, copies = _fork(sched, seq)
    bm = sched.block_manager
    assert child.block_table[:2] == seq.block_table[:2] and copies == [(seq.block_table[2], child.block_table[2], 2)]
    assert [bm.blocks[b].ref_count for b in seq.block_table] == [2, 2, 1]
    assert child.num_computed_tokens == 10 and child.gap == 1 and child.status == SequenceStatus.RUNNING
    for _ in range(5):  # both decode on, each in its own blocks
        batch = sched.schedule()
        assert {s.seq_id for s in batch} == {seq.seq_id, child.seq_id}
        sched.postprocess(batch, [8, 9])
    assert seq.block_table[2:] != child.block_table[2:] and not set(seq.block_table[2:]) & set(child.block_table[2:])
    sched.preempt(child)
    assert [bm.blocks[b].ref_count for b in seq.block_table[:2]] == [1, 1]
    sched.block_manager.deallocate(seq)
    assert bm.free_blocks_nums == 8 and not bm.used_blocks


def test_fork_at_a_page_border_copies_nothing():
    sched = Scheduler(2, 4, max_num_seqs=4)
    seq = _running(sched, 8)
    child, copies = _fork(sched, seq)  # no free block is needed yet
    assert copies == [] and child.block_table == seq.block_table


def test_fork_refusals_change_nothing():
    sched = Scheduler(3, 4, max_num_seqs=2)
    queued = Sequence([1, 2, 3])
    with pytest.raises(ValueError, match="not running"):
        _fork(sched, queued)
    seq = _running(sched, 10)
    with pytest.raises(RuntimeError, match="no free KV block"):
        _fork(sched, seq)
    assert [sched.block_manager.blocks[b].ref_count for b in seq.block_table] == [1, 1, 1]
    assert list(sched.running) == [seq]
    sched = Scheduler(8, 4, max_num_seqs=1)
    seq = _running(sched, 10)
    with pytest.raises(RuntimeError, match="max_num_seqs"):
        _fork(sched, seq)


def test_config_takes_the_4bit_cache():
    from microserve_b200.Config import Config
    assert Config(kv_cache_dtype="fp4_e2m1").kv_cache_dtype == "fp4_e2m1"
    with pytest.raises(AssertionError):
        Config(kv_cache_dtype="fp4_e2m1", dtype=torch.bfloat16)
