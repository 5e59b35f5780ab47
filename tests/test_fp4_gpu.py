"""The 4-bit KV cache and page copies on the GPU against the 64-bit oracle (oracle/fp4_kv.py).

Codes, scales, loaded values and copied pages: bit-exact. Attention: with o the exact
output and A = sum p |v| (both 64-bit), an output may be off by
  2^-11 |o|   its own rounding to fp16 (plus 2^-25 below the normal range), and
  A * (2^-12 + d): d = 2^-13 for what fp32 leaves: a score is a sum of 128 exact products,
  off by at most 128 * 2^-24 of sum |q k| scale <= 60 here, times ln-to-log2 and exp2's own
  2^-22, below 2^-13; the sums over up to 2^12 keys add 2^-12 at worst (2^-24 per addition);
  prefill may round each weight to fp16: another 2^-11.
"""
import pytest
import torch

from oracle import fp4_kv as F

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 128 ** -0.5


@pytest.fixture(autouse=True)
def _status_clean():
    from microserve_b200 import _lib
    _lib.load()
    yield
    assert _lib.device_status() == 0, "a kernel recorded a status that the test did not take"


def _close(got, o, a, prefill=False):
    err = (got.cpu().double() - o).abs()
    tol = o.abs() * 2.0 ** -11 + 2.0 ** -25 + a * (2.0 ** -12 + 2.0 ** -13 + (2.0 ** -11 if prefill else 0))
    worst = ((err - tol).max()).item()
    assert torch.isfinite(got).all() and worst <= 0, (worst, err.max().item())


def _cache(NB, BS, H, seed, fill="data"):
    """(codes, scales) of K and V on the CPU: quantised random data, or bytes that no read may let through."""
    g = torch.Generator().manual_seed(seed)
    if fill == "poison":  # NaN scales everywhere
        codes = torch.randint(0, 256, (2, NB, H, BS, 64), generator=g, dtype=torch.uint8)
        scales = torch.full((2, NB, H, BS, 8), 255, dtype=torch.uint8)
    else:
        x = torch.randn(2, NB, H, BS, 128, generator=g).half()
        x[..., 5] *= 8
        codes, scales = F.encode(x)
    return [codes[0].clone(), codes[1].clone(), scales[0].clone(), scales[1].clone()]


def _dev(c):
    return [t.to(DEV) for t in c]


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _tables(lens, BS, seed, extra=2, width=None):
    """Random distinct pages per sequence, -1 behind them; (tables, number of pages)."""
    need = [(n + BS - 1) // BS for n in lens]
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(sum(need) + extra, generator=g).tolist()
    w = width or max(max(need), 1)
    t = torch.full((len(lens), w), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = torch.tensor(perm[at:at + n], dtype=torch.int32)
        at += n
    return t, sum(need) + extra


# ------------------------------------------------------------------ store, load
@pytest.mark.parametrize("T,H,BS", [(1, 1, 64), (1, 8, 256), (3, 8, 256), (17, 3, 192), (300, 2, 64), (77, 5, 512)])
def test_store_and_load_bit_exact(T, H, BS):
    from microserve_b200 import kernels
    g = torch.Generator().manual_seed(T + H)
    NB = T // BS + 2
    c = _cache(NB, BS, H, 1)
    d = _dev(c)
    qkv = (torch.randn(T, (4 + 2 * H) * 128, generator=g) * torch.exp2(torch.randint(-20, 12, (T, 1), generator=g)))
    qkv = qkv.clamp(-65504, 65504).half()
    qkv[0, 4 * 128:4 * 128 + 32] = 0
    qkv[0, 4 * 128 + 3] = -0.0
    k, v = (qkv[:, a * 128:(a + H) * 128].unflatten(1, (H, 128)) for a in (4, 4 + H))  # slices of the projection
    slots = torch.randperm(NB * BS, generator=g)[:T]
    if T > 2:
        slots[1] = -1
    F.store(k, v, *c, slots)
    dq = qkv.to(DEV)
    dk, dv = (dq[:, a * 128:(a + H) * 128].unflatten(1, (H, 128)) for a in (4, 4 + H))
    kernels.store_kv_fp4(dk, dv, *d, slots.to(DEV))
    for got, ref in zip(d, c):  # every byte: the rows stored, and the ones that were there
        assert torch.equal(got.cpu(), ref)
    lk, lv = kernels.load_kv_fp4(*d, slots.to(DEV))
    s = slots.clamp_min(0)
    for got, codes, scales in ((lk, c[0], c[2]), (lv, c[1], c[3])):
        ref = F.decode(codes[s // BS, :, s % BS], scales[s // BS, :, s % BS])
        ref = torch.where((slots >= 0)[:, None, None], ref, torch.zeros_like(ref))
        assert torch.equal(got.cpu().double(), ref)


def test_store_every_fp16_value_bit_exact():
    """All 65536 fp16 bit patterns (NaNs and infinities among them), each in a group whose other elements are
    smaller, and again beside a larger element: every rounding point of codes and scales."""
    from microserve_b200 import kernels
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    small = x.repeat_interleave(128).view(-1, 128).clone()  # [65536, 128]: 8 groups a pattern
    f = small.float().view(-1, 8, 16)
    mult = torch.linspace(0, 1, 16).view(1, 1, 16) * torch.tensor([1, .5, .25, .75, .9, .1, -1, .6]).view(1, 8, 1)
    y = torch.where(f.isfinite(), f * mult, f).clamp(-65504, 65504).half()
    y[..., 15] = x.view(-1, 1)
    z = torch.where(f.isfinite(), f / torch.tensor([8, 3, 1.7, 1.2, 1, 2, 5, 6]).view(1, 8, 1), f).half()
    z[:, :, 0] = x.view(-1, 1)
    k, v = y.view(-1, 128, 128)[:, :, :], z.view(-1, 128, 128)  # [512 tokens, 128 heads, 128]
    NB, BS = 8, 64
    codes, scales = torch.zeros(NB, 128, BS, 64, dtype=torch.uint8), torch.zeros(NB, 128, BS, 8, dtype=torch.uint8)
    c = [codes, codes.clone(), scales, scales.clone()]
    d = _dev(c)
    slots = torch.arange(512)
    F.store(k, v, *c, slots)
    kernels.store_kv_fp4(k.to(DEV), v.to(DEV), *d, slots.to(DEV))
    for got, ref in zip(d, c):
        assert torch.equal(got.cpu(), ref)
    lk, _ = kernels.load_kv_fp4(*d, slots.to(DEV))
    ref = F.decode(*(t[slots // BS, :, slots % BS] for t in (c[0], c[2])))
    assert torch.equal(lk.cpu().double().nan_to_num(7.25), ref.nan_to_num(7.25))


def test_unaligned_single_and_expanded_inputs():
    """One token with any stride, rows that are not 16-byte vectors, a head broadcast over all heads."""
    from microserve_b200 import kernels
    BS, H = 64, 2
    base = torch.randn(6, H * 128 + 3, generator=torch.Generator().manual_seed(3)).half()
    odd = base[:, 1:1 + H * 128].unflatten(1, (H, 128))
    one = base.t()[:256, :1].t().unflatten(1, (H, 128))
    wide = base[:, :128].unsqueeze(1).expand(6, H, 128)
    for k in (odd, one, wide):
        T = k.shape[0]
        c = _cache(2, BS, H, 5)
        d = _dev(c)
        slots = torch.arange(T)
        F.store(k, k, *c, slots)
        kk = base.to(DEV)
        kk = (kk[:, 1:1 + H * 128].unflatten(1, (H, 128)) if k is odd else
              kk.t()[:256, :1].t().unflatten(1, (H, 128)) if k is one else kk[:, :128].unsqueeze(1).expand(6, H, 128))
        kernels.store_kv_fp4(kk, kk, *d, slots.to(DEV))
        assert all(torch.equal(a.cpu(), b) for a, b in zip(d, c))


def test_slots_outside_the_cache_are_skipped_and_recorded():
    from microserve_b200 import _lib, kernels
    c = _cache(2, 64, 2, 9)
    d = _dev(c)
    x = torch.randn(3, 2, 128, generator=torch.Generator().manual_seed(1)).half().to(DEV)
    slots = torch.tensor([128, 5, 1 << 40], device=DEV)
    kernels.store_kv_fp4(x, x, *d, slots)
    F.store(x.cpu(), x.cpu(), *c, torch.tensor([-1, 5, -1]))
    assert all(torch.equal(a.cpu(), b) for a, b in zip(d, c))
    assert _lib.device_status() == 3 and _lib.device_status() == 0
    k, _ = kernels.load_kv_fp4(*d, slots)
    assert (k[0] == 0).all() and (k[2] == 0).all() and (k[1] != 0).any() and _lib.device_status() == 3


# ------------------------------------------------------------------ decode
DECODE = [
    ([1], 16, 8, 256), ([300], 16, 8, 256), ([0, 5, 0, 64], 8, 8, 64), ([63, 65, 128, 1, 0, 191, 193], 12, 4, 64),
    ([257, 1000, 3, 511], 32, 8, 256), ([700, 1], 64, 8, 192), ([33, 900], 7, 1, 128), ([40, 1300], 10, 2, 512),
    ([2900], 8, 1, 256), ([31, 32, 33], 6, 1, 64), ([4090, 17], 5, 1, 128),
]


@pytest.mark.parametrize("lens,Hq,Hkv,BS", DECODE)
@pytest.mark.parametrize("width", [None, 33])
def test_decode_vs_oracle(lens, Hq, Hkv, BS, width):
    from microserve_b200 import kernels
    need = max((n + BS - 1) // BS for n in lens)
    if width is not None and width < need:
        width = need + 30
    bt, NB = _tables(lens, BS, 2, width=width)
    c = _cache(NB, BS, Hkv, 3)
    for b, n in enumerate(lens):  # what lies behind a sequence's end must not matter
        if n % BS:
            page = int(bt[b, n // BS])
            for t in c[2:]:
                t[page, :, n % BS:] = 255
    q = (torch.randn(len(lens), Hq + 2, 128, generator=torch.Generator().manual_seed(4)) * 2).half()[:, 1:1 + Hq]
    o, a = F.decode_attention(q, *c, lens, bt, SCALE)
    dq = torch.zeros(len(lens), Hq + 2, 128, dtype=torch.float16, device=DEV)
    dq[:, 1:1 + Hq] = q.to(DEV)
    got = kernels.paged_decode_fp4(dq[:, 1:1 + Hq], *_dev(c), _i32(lens), bt.to(DEV), SCALE)  # strided rows
    _close(got, o, a)
    assert all((got[b] == 0).all() for b, n in enumerate(lens) if n == 0)


def test_decode_bad_pages_and_lengths():
    """Pages outside the cache count as masked, a length past the table is cut; both are recorded."""
    from microserve_b200 import _lib, kernels
    BS, lens = 64, [200, 200, 100, 64]
    bt, NB = _tables(lens, BS, 8, width=4)
    c = _cache(NB, BS, 2, 8)
    q = torch.randn(4, 4, 128, generator=torch.Generator().manual_seed(4)).half()
    bad = bt.clone()
    bad[0, 1] = -1
    bad[1, 0] = NB
    bad[3, 0] = 1 << 30
    got = kernels.paged_decode_fp4(q.to(DEV), *_dev(c), _i32(lens), bad.to(DEV), SCALE)
    assert _lib.device_status() == 3
    # the same with the tokens of those pages left out
    for b, cols, n in ((0, [0, 2, 3], 136), (1, [1, 2, 3], 136), (2, [0, 1], 100)):
        t = bt[b, cols]
        k, v = F.gather(c[0], c[2], t, n), F.gather(c[1], c[3], t, n)
        for h in range(4):
            p = torch.softmax(q[b, h].double() @ k[h // 2].t() * SCALE, -1)
            _close(got[b, h], p @ v[h // 2], p @ v[h // 2].abs())
    assert (got[3] == 0).all()
    over = kernels.paged_decode_fp4(q.to(DEV), *_dev(c), _i32([5000, 2**31 - 1, 3, -7]), bt.to(DEV), SCALE)
    assert _lib.device_status() == 3
    assert torch.isfinite(over[2]).all() and (over[3] == 0).all()


def test_nan_and_inf_reach_only_their_own_rows():
    from microserve_b200 import kernels
    BS, lens = 64, [100, 100, 100]
    bt, NB = _tables(lens, BS, 5)
    c = _cache(NB, BS, 2, 5)
    q = torch.randn(3, 4, 128, generator=torch.Generator().manual_seed(4)).half()
    q[0, 0, 3] = float("nan")
    c[2][int(bt[1, 0]), 1, 7, 2] = 255  # a NaN among the keys of kv head 1 of sequence 1
    c[3][int(bt[2, 1]), 0, 3, 7] = 255  # and among the values of kv head 0 of sequence 2 (elements 112..127)
    got = kernels.paged_decode_fp4(q.to(DEV), *_dev(c), _i32(lens), bt.to(DEV), SCALE).cpu()
    nan = torch.zeros_like(got, dtype=torch.bool)
    nan[0, 0] = nan[1, 2:] = True
    nan[2, :2, 112:] = True
    assert torch.equal(got.isnan(), nan)


def test_large_scores_and_equal_scores():
    """Scores far apart (one key takes all the weight), all equal, and of the largest magnitudes."""
    from microserve_b200 import kernels
    BS, n = 64, 150
    bt, NB = _tables([n, n, n], BS, 6)
    c = _cache(NB, BS, 1, 6)
    q = torch.randn(3, 1, 128, generator=torch.Generator().manual_seed(1)).half()
    q[0] *= 40
    q[1] = 0
    q[2] = 60000
    ks = c[2].clone()
    o, a = F.decode_attention(q, c[0], c[1], ks, c[3], [n, n, n], bt, SCALE)
    got = kernels.paged_decode_fp4(q.to(DEV), *_dev(c), _i32([n, n, n]), bt.to(DEV), SCALE)
    _close(got[1], o[1], a[1])
    # row 0: scores up to ~500: their fp32 sums are off by up to 2^-17 of sum |q k| scale ~ 400 * 128 / 11.3: 0.04
    err = (got[0].cpu().double() - o[0]).abs()
    assert (err <= o[0].abs() * 2.0 ** -11 + 0.08 * a[0] + 2.0 ** -25).all()
    assert torch.isfinite(got).all()


def test_offsets_past_32_bits():
    """Pages whose byte offsets pass 2^32: codes of 41000 pages of 8 heads."""
    from microserve_b200 import kernels
    NB, BS, H = 41000, 256, 8
    d = [torch.zeros(NB, H, BS, w, dtype=torch.uint8, device=DEV) for w in (64, 64, 8, 8)]
    pages = [40999, 3, 33000]
    c = _cache(3, BS, H, 7)
    for t, s in zip(d, c):
        t[pages] = s.to(DEV)
    n, Hq = 600, 16
    q = torch.randn(1, Hq, 128, generator=torch.Generator().manual_seed(2)).half()
    o, a = F.decode_attention(q, *c, [n], torch.tensor([[0, 1, 2]]), SCALE)
    got = kernels.paged_decode_fp4(q.to(DEV), *d, _i32([n]), _i32([pages]), SCALE)
    _close(got, o, a)
    got = kernels.paged_prefill_fp4(q.to(DEV), *d, _i32([pages]), _i32([0, 1]), _i32([n]), SCALE)
    _close(got, o, a, prefill=True)
    x = torch.randn(2, H, 128, generator=torch.Generator().manual_seed(3)).half()
    slots = torch.tensor([40999 * BS + 255, 33000 * BS + 1])
    kernels.store_kv_fp4(x.to(DEV), x.to(DEV), *d, slots.to(DEV))
    k, _ = kernels.load_kv_fp4(*d, slots.to(DEV))
    assert torch.equal(k.cpu().double(), F.decode(*F.encode(x)))


# ------------------------------------------------------------------ prefill
PREFILL = [  # (q_len, prefix) per sequence
    ([(1, 0)], 16, 8, 256), ([(8, 292), (8, 692)], 16, 8, 256), ([(130, 0), (0, 50), (3, 61)], 8, 8, 64),
    ([(33, 200), (64, 64), (1, 127)], 12, 4, 64), ([(257, 130)], 32, 8, 256), ([(100, 1000)], 64, 8, 192),
    ([(19, 700), (40, 3)], 7, 1, 128), ([(70, 500), (0, 0), (65, 0)], 10, 2, 512), ([(300, 1)], 8, 1, 256),
    ([(2, 1500)], 6, 1, 64), ([(128, 384), (129, 383)], 5, 1, 128), ([(16, 40)], 4, 4, 64), ([(600, 100)], 4, 1, 128),
]


@pytest.mark.parametrize("seqs,Hq,Hkv,BS", PREFILL)
def test_prefill_vs_oracle(seqs, Hq, Hkv, BS):
    from microserve_b200 import kernels
    kv = [q + p for q, p in seqs]
    bt, NB = _tables(kv, BS, 2)
    c = _cache(NB, BS, Hkv, 3)
    for b, n in enumerate(kv):
        if n % BS:
            page = int(bt[b, n // BS])
            for t in c[2:]:
                t[page, :, n % BS:] = 255
    cu = [0]
    for n, _ in seqs:
        cu.append(cu[-1] + n)
    T = cu[-1] + 5  # rows behind the last sequence
    q = (torch.randn(T, Hq, 128, generator=torch.Generator().manual_seed(4)) * 2).half()
    o, a = F.prefill_attention(q, *c, bt, cu, kv, SCALE)
    out = torch.full((T, Hq, 128), 3.25, dtype=torch.float16, device=DEV)
    got = kernels.paged_prefill_fp4(q.to(DEV), *_dev(c), bt.to(DEV), _i32(cu), _i32(kv), SCALE, out=out)
    assert got is out and (out[cu[-1]:] == 3.25).all()
    _close(got[:cu[-1]], o, a, prefill=True)


def test_prefill_queries_without_keys_bad_pages_and_lengths():
    """Queries at negative positions give 0; bad pages count as masked; a length past the table is cut."""
    from microserve_b200 import _lib, kernels
    BS, H = 64, 2
    bt, NB = _tables([200, 200, 200], BS, 8, width=4)
    c = _cache(NB, BS, H, 8)
    q = torch.randn(36, 4, 128, generator=torch.Generator().manual_seed(4)).half()
    cu, kv = [0, 12, 24, 36], [5, 0, 200]
    got = kernels.paged_prefill_fp4(q.to(DEV), *_dev(c), bt.to(DEV), _i32(cu), _i32(kv), SCALE)
    o, a = F.prefill_attention(q, *c, bt, cu, kv, SCALE)
    assert (got[:7] == 0).all() and (got[12:24] == 0).all()
    _close(got, o, a, prefill=True)
    bad = bt.clone()
    bad[0, 0], bad[2, 1], bad[2, 3] = NB, -1, -5
    got = kernels.paged_prefill_fp4(q.to(DEV), *_dev(c), bad.to(DEV), _i32(cu), _i32(kv), SCALE)
    assert _lib.device_status() == 3
    assert (got[:24] == 0).all()
    k, v = (torch.cat([F.gather(x, s, bt[2], 200)[:, :64], F.gather(x, s, bt[2], 200)[:, 128:192]], 1)
            for x, s in ((c[0], c[2]), (c[1], c[3])))
    for i, h in ((8, 0), (11, 3)):  # queries at 196 and 199 see all of pages 0 and 2
        p = torch.softmax(q[24 + i, h].double() @ k[h // 2].t() * SCALE, -1)
        _close(got[24 + i, h], p @ v[h // 2], p @ v[h // 2].abs(), prefill=True)
    got = kernels.paged_prefill_fp4(q.to(DEV), *_dev(c), bt.to(DEV), _i32(cu), _i32([5, 2**31 - 1, 9000]), SCALE)
    assert _lib.device_status() == 3


def test_prefill_nan_reaches_only_its_own_rows():
    from microserve_b200 import kernels
    BS = 64
    bt, NB = _tables([150], BS, 5)
    c = _cache(NB, BS, 2, 5)
    q = torch.randn(40, 4, 128, generator=torch.Generator().manual_seed(4)).half()
    q[7, 0, 3] = float("nan")
    c[2][int(bt[0, 2]), 1, 2, 4] = 255  # key 130 of kv head 1: queries 20.. see it
    c[3][int(bt[0, 2]), 0, 12, 0] = 255  # value 140 of kv head 0, elements 0..15: queries 30.. see it
    got = kernels.paged_prefill_fp4(q.to(DEV), *_dev(c), bt.to(DEV), _i32([0, 40]), _i32([150]), SCALE).cpu()
    nan = torch.zeros_like(got, dtype=torch.bool)
    nan[7, 0] = True
    nan[20:, 2:] = True
    nan[30:, :2, :16] = True
    assert torch.equal(got.isnan(), nan)


# ------------------------------------------------------------------ copies
@pytest.mark.parametrize("kind", ["fp8", "fp4"])
@pytest.mark.parametrize("L,H,BS,n,part", [(1, 1, 64, 1, False), (3, 8, 256, 5, True), (2, 5, 64, 9, True),
                                           (4, 2, 192, 3, False)])
def test_copy_pages(kind, L, H, BS, n, part):
    from microserve_b200 import kernels
    g = torch.Generator().manual_seed(n)
    NB = 2 * n + 1
    if kind == "fp8":
        cache = torch.randint(0, 256, (2, L, NB, BS, H, 128), generator=g, dtype=torch.uint8).view(torch.float8_e4m3fn)
        scale = torch.rand(2, L, NB, BS, H, generator=g)
    else:
        cache = torch.randint(0, 256, (2, L, NB, H, BS, 64), generator=g, dtype=torch.uint8)
        scale = torch.randint(0, 256, (2, L, NB, H, BS, 8), generator=g, dtype=torch.uint8)
    ids = torch.randperm(NB, generator=g).tolist()
    src, dst = [ids[i // 2] for i in range(n)], ids[n:2 * n]  # a page may be copied twice
    tok = [[0, 1, 3, BS - 1, BS, BS + 7, -2][i % 7] for i in range(n)] if part else None
    rc, rs = cache.clone().view(torch.uint8), scale.clone()
    for i in range(n):
        m = min(max(tok[i], 0), BS) if part else BS
        for r in (rc, rs):
            a, b = (r[:, :, src[i]], r[:, :, dst[i]])
            if kind == "fp8":
                b[:, :, :m] = a[:, :, :m]
            else:
                b[:, :, :, :m] = a[:, :, :, :m]
    dc, ds = cache.to(DEV), scale.to(DEV)
    kernels.copy_pages(dc, ds, _i32(src), _i32(dst), _i32(tok) if part else None)
    assert torch.equal(dc.view(torch.uint8).cpu(), rc) and torch.equal(ds.cpu(), rs)
    # one layer's K alone: a view without planes
    one = cache[0, L - 1].clone().to(DEV), scale[0, L - 1].clone().to(DEV)
    kernels.copy_pages(*one, _i32(src), _i32(dst), _i32(tok) if part else None)
    assert torch.equal(one[0].view(torch.uint8).cpu(), rc[0, L - 1]) and torch.equal(one[1].cpu(), rs[0, L - 1])


def test_copy_pages_outside_the_cache_are_skipped():
    from microserve_b200 import _lib, kernels
    c = _cache(4, 64, 2, 9)
    d = _dev(c)
    kernels.copy_pages(d[0], d[2], _i32([0, -1, 4, 1, 2]), _i32([3, 1, 1, 4, 2]))
    assert _lib.device_status() == 3
    ref = c[0].clone()
    ref[3] = ref[0]
    assert torch.equal(d[0].cpu(), ref)


# ------------------------------------------------------------------ together, graphs, streams
def test_cache_run_store_prefill_fork_decode():
    """A prompt stored and attended to in two chunks, its last page forked, then both branches decode with
    different tokens: each against the oracle on its own cache."""
    from microserve_b200 import kernels
    BS, H, Hq, n = 64, 2, 8, 150
    g = torch.Generator().manual_seed(12)
    k, v = (torch.randn(n + 8, H, 128, generator=g).half() for _ in range(2))
    q = torch.randn(n + 8, Hq, 128, generator=g).half()
    c = _cache(8, BS, H, 0, fill="poison")
    d = _dev(c)
    table = [6, 1, 4]
    bt = torch.tensor([table], dtype=torch.int32)
    for a, b in ((0, 90), (90, n)):
        slots = torch.tensor([table[p // BS] * BS + p % BS for p in range(a, b)])
        F.store(k[a:b], v[a:b], *c, slots)
        kernels.store_kv_fp4(k[a:b].to(DEV), v[a:b].to(DEV), *d, slots.to(DEV))
        got = kernels.paged_prefill_fp4(q[a:b].to(DEV), *d, bt.to(DEV), _i32([0, b - a]), _i32([b]), SCALE)
        o, s = F.prefill_attention(q[a:b], *c, bt, [0, b - a], [b], SCALE)
        _close(got, o, s, prefill=True)
    both = [torch.stack((d[0], d[1])), torch.stack((d[2], d[3]))]
    kernels.copy_pages(both[0], both[1], _i32([4]), _i32([2]), _i32([n % BS]))
    d = [both[0][0], both[0][1], both[1][0], both[1][1]]
    for t in c:
        t[2, :, :n % BS] = t[4, :, :n % BS]
    tables = [table, [6, 1, 2]]
    bt = torch.tensor(tables, dtype=torch.int32)
    for step in range(4):
        p = n + step
        slots = torch.tensor([t[p // BS] * BS + p % BS for t in tables])
        rows = torch.tensor([p, p + 4])
        F.store(k[rows], v[rows], *c, slots)
        kernels.store_kv_fp4(k[rows].to(DEV), v[rows].to(DEV), *d, slots.to(DEV))
        got = kernels.paged_decode_fp4(q[rows].to(DEV), *d, _i32([p + 1] * 2), bt.to(DEV), SCALE)
        _close(got, *F.decode_attention(q[rows], *c, [p + 1] * 2, bt, SCALE))
    assert all(torch.equal(a.cpu(), b) for a, b in zip(d, c))


def test_captured_graphs_and_streams():
    """Two captured graphs of different batches replayed in turn with new lengths, and the same calls at once on
    two streams: every result as the eager one."""
    from microserve_b200 import kernels
    BS, H, Hq = 64, 2, 8
    lens = [[700, 3, 0, 129], [64, 1900]]
    runs = []
    for i, ls in enumerate(lens):
        bt, NB = _tables(ls, BS, i, width=40)
        c = _dev(_cache(NB, BS, H, i))
        q = torch.randn(len(ls), Hq, 128, generator=torch.Generator().manual_seed(i)).half().to(DEV)
        runs.append([q, c, _i32(ls), bt.to(DEV)])
    call = lambda r: kernels.paged_decode_fp4(r[0], *r[1], r[2], r[3], SCALE)  # noqa: E731
    pre = lambda r: kernels.paged_prefill_fp4(r[0][:2], *r[1], r[3][1:2], _i0, r[2][1:2], SCALE)  # noqa: E731
    _i0 = _i32([0, 2])
    eager = [(call(r), pre(r)) for r in runs]
    graphs = []
    for r in runs:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call(r), pre(r)
        graphs.append((g, out))
    for order in ((0, 1, 0), (1, 0, 1)):
        for i in order:
            graphs[i][0].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(graphs[i][1], eager[i]))
    runs[0][2].copy_(_i32([70, 64, 0, 1]))
    want = call(runs[0])
    graphs[0][0].replay()
    assert torch.equal(graphs[0][1][0], want)
    runs[0][2].copy_(_i32(lens[0]))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append((call(runs[i]), pre(runs[i])))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for o in outs[i] for a, b in zip(o, eager[i]))


# ------------------------------------------------------------------ engine
def _engine(kind, eager, **kw):
    from microserve_b200.Config import Config
    from microserve_b200.engine.llm import LLMEngine
    from tests.model_utils import qwen3_config
    return LLMEngine(Config(hf_config=qwen3_config(layers=2), load_format="dummy", enforce_eager=eager,
                            num_kvcache_blocks=12, max_num_seqs=4, max_model_len=1024, max_num_batched_tokens=200,
                            seed=0, kv_cache_dtype=kind, **kw))


def test_engine_on_the_4bit_cache(monkeypatch):
    """LLMEngine with kv_cache_dtype="fp4_e2m1": chunked prefill and decode; every attention call of the eager run
    against the oracle on the engine's own cache, the captured graphs' tokens equal to the eager ones."""
    from microserve_b200 import kernels
    from microserve_b200.engine.sequence import SamplingParams
    prompts = [torch.randint(100, 4096, (n,), generator=torch.Generator().manual_seed(n)).tolist() for n in (300, 45)]
    seen = {"decode": 0, "prefill": 0}
    decode, prefill = kernels.paged_decode_fp4, kernels.paged_prefill_fp4

    def check_decode(q, kc, vc, ks, vs, lens, bt, scale, out=None):
        got = decode(q, kc, vc, ks, vs, lens, bt, scale, out=out)
        _close(got, *F.decode_attention(q.cpu(), kc.cpu(), vc.cpu(), ks.cpu(), vs.cpu(), lens.tolist(), bt.cpu(),
                                        scale))
        seen["decode"] += 1
        return got

    def check_prefill(q, kc, vc, ks, vs, bt, cu, kv, scale, out=None):
        got = prefill(q, kc, vc, ks, vs, bt, cu, kv, scale, out=out)
        _close(got, *F.prefill_attention(q.cpu(), kc.cpu(), vc.cpu(), ks.cpu(), vs.cpu(), bt.cpu(), cu.tolist(),
                                         kv.tolist(), scale), prefill=True)
        seen["prefill"] += 1
        return got

    tokens = []
    for eager in (True, False):
        with monkeypatch.context() as m:
            if eager:
                m.setattr(kernels, "paged_decode_fp4", check_decode)
                m.setattr(kernels, "paged_prefill_fp4", check_prefill)
            eng = _engine("fp4_e2m1", eager)
            seqs = [eng.add(p, SamplingParams(temperature=0.0), max_tokens=8) for p in prompts]
            while not eng.is_idle():
                eng.step()
        assert eng.runner.kv_cache.dtype == torch.uint8 and all(len(s.completion_token_ids) == 8 for s in seqs)
        tokens.append([s.completion_token_ids for s in seqs])
        if not eager:
            eng.runner.release_graphs()
    assert tokens[0] == tokens[1]
    assert seen["decode"] >= 2 * 7 and seen["prefill"] >= 2


@pytest.mark.parametrize("kind", ["fp8_e4m3", "fp4_e2m1"])
def test_engine_fork(kind):
    """A greedy fork continues as its parent does (each from its own last page), and as the same engine does
    without a fork; a fork at a page border too."""
    from microserve_b200.engine.sequence import SamplingParams
    greedy = SamplingParams(temperature=0.0)
    for n in (77, 250):  # 250: the fork comes after 6 steps, at 256 computed tokens
        prompt = torch.randint(100, 4096, (n,), generator=torch.Generator().manual_seed(n)).tolist()
        alone = _engine(kind, True).generate(prompt, greedy, max_tokens=20)
        eng = _engine(kind, True)
        seq = eng.add(prompt, greedy, max_tokens=20)
        while seq.num_computed_tokens < (256 if n == 250 else n + 4):
            eng.step()
        child = eng.fork(seq)
        hot = eng.fork(seq, SamplingParams(temperature=1.5), max_tokens=15)
        while not eng.is_idle():
            eng.step()
        assert seq.completion_token_ids == alone == child.completion_token_ids
        assert len(hot.completion_token_ids) == 15 and eng.scheduler.block_manager.free_blocks_nums == 12
        with pytest.raises(ValueError, match="not running"):
            eng.fork(seq)
