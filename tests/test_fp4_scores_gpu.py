"""The attentions over the 4-bit KV cache where scores climb, fall and jump along a sequence, so that the softmax
reference moves and what was summed is rescaled, and where scores are of the largest magnitudes.

Only element 0 of the queries and keys is not zero in the first tests, and it has few bits, so a score is exact in
fp32. With o the exact output and A = sum p |v|, an output may be off by its own rounding, 2^-11 |o| + 2^-25, and by
A * (2^-12 + 2^-13): 2^-12 for the sums over up to 2^12 keys (2^-24 an addition), 2^-13 for the rest: a reference
of up to 1200 in the log2 domain is rounded by 2^-24 * 1200 < 2^-13 / 1.4, and so is each of the two in a rescale, but what
a rescale leaves of earlier sums is at most 2^-5 of them, exp2's own error is 2^-22, and the scale's two
roundings count for the at most 2^5 that a key with any weight lies below the largest. Prefill rounds weights to f16:
another 2^-11 A (half a step), and 2^-31 of max |v| for each key whose weight is subnormal there (half a step of 2^-24,
the largest weight being 2^6 or more).
"""
import pytest
import torch

from oracle import fp4_kv as F
from tests.test_fp4_gpu import DEV, SCALE, _dev, _i32, _status_clean, _tables  # noqa: F401

pytestmark = pytest.mark.gpu

STEP = 64
# height of key t in units of about one in the log2 domain, for a query of 8
SHAPES = {
    "rising": lambda t: 12.0 * (t // STEP),
    "slowly": lambda t: 0.09 * t,
    "falling": lambda t: 600.0 - 12.0 * (t // STEP),
    "alternating": lambda t: 25.0 * ((t // STEP) % 2) + 3.0 * (t // STEP),
    "late": lambda t: 300.0 * (t >= (t.max() * 4) // 5),
    "spikes": lambda t: 40.0 * (t % 97 == 5) + 0.5 * (t // 32),
}
QUERIES = (8.0, -8.0, 4.0, 16.0, 0.0, 2.0, -1.0, 0.5)


def _climbing(lens, BS, Hkv, shape, seed):
    """(block tables, cache): keys of one element with the heights of `shape`, random values."""
    g = torch.Generator().manual_seed(seed)
    bt, NB = _tables(lens, BS, seed)
    k = torch.zeros(NB, BS, Hkv, 128, dtype=torch.float16)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        t = torch.arange(n)
        x = SHAPES[shape](t).double()[:, None] + 4 * torch.rand(n, Hkv, generator=g).double()
        k[bt[b].long()[t // BS], t % BS, :, 0] = x.half()
    v = torch.randn(NB, BS, Hkv, 128, generator=g).half()
    (kc, ks), (vc, vs) = (F.encode(x.transpose(1, 2).contiguous()) for x in (k, v))
    return bt, [kc, vc, ks, vs]


def _one_element(T, Hq, values=QUERIES):
    q = torch.zeros(T, Hq, 128, dtype=torch.float16)
    q[..., 0] = torch.tensor(values)[(torch.arange(T)[:, None] * 3 + torch.arange(Hq)) % len(values)].half()
    return q


def _within(got, o, a, keys=None, vmax=0.0):
    """keys: the most that a row sees, for prefill; None for decode."""
    err = (got.cpu().double() - o).abs()
    tol = o.abs() * 2.0 ** -11 + 2.0 ** -25 + a * (2.0 ** -12 + 2.0 ** -13)
    if keys is not None:
        tol = tol + a * 2.0 ** -11 + keys * 2.0 ** -31 * vmax
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), ((err - tol).max().item(), err.max().item())


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("lens,Hq,Hkv,BS", [
    ([3000], 4, 1, 64),                          # every CTA has a piece of one item
    ([2900, 65, 0, 1500, 64], 16, 2, 128),       # 8 heads a kv head
    ([700] * 40 + [31, 33], 32, 8, 256),         # items inside a warp's share, and across warps
    ([1900, 1100], 5, 1, 192),
])
def test_decode_with_moving_references(shape, lens, Hq, Hkv, BS):
    from microserve_b200 import kernels
    bt, c = _climbing(lens, BS, Hkv, shape, 21)
    q = _one_element(len(lens), Hq)
    args = (q.to(DEV), *_dev(c), _i32(lens), bt.to(DEV), SCALE)
    got = kernels.paged_decode_fp4(*args)
    _within(got, *F.decode_attention(q, *c, lens, bt, SCALE))
    for _ in range(5):
        assert torch.equal(kernels.paged_decode_fp4(*args), got)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("seqs,Hq,Hkv,BS", [
    ([(40, 2960)], 8, 1, 64),                    # one item over many CTAs, a few steps each
    ([(70, 1500)] * 6 + [(3, 100)], 32, 8, 256),  # CTAs with long runs of steps and items cut by shares
    ([(500, 0), (129, 700)], 4, 4, 128),         # rows of one tile that see 1 to 500 keys
    ([(90, 1900)], 14, 2, 192),
])
def test_prefill_with_moving_references(shape, seqs, Hq, Hkv, BS):
    from microserve_b200 import kernels
    kv = [q + p for q, p in seqs]
    cu = [0]
    for n, _ in seqs:
        cu.append(cu[-1] + n)
    bt, c = _climbing(kv, BS, Hkv, shape, 22)
    q = _one_element(cu[-1], Hq)
    args = (q.to(DEV), *_dev(c), bt.to(DEV), _i32(cu), _i32(kv), SCALE)
    got = kernels.paged_prefill_fp4(*args)
    o, a = F.prefill_attention(q, *c, bt, cu, kv, SCALE)
    _within(got, o, a, max(kv), F.decode(c[1], c[3]).abs().max().item())
    for _ in range(5):
        assert torch.equal(kernels.paged_prefill_fp4(*args), got)


# ------------------------------------------------------------------ the largest magnitudes
def _filled(n, BS, k, seed):
    """(block table, cache, fp64 values [n, 128]) of one sequence and kv head with keys k [n, 128]."""
    bt, NB = _tables([n], BS, seed)
    t = torch.arange(n)
    g = torch.Generator().manual_seed(seed)
    kk, vv = torch.zeros(NB, 1, BS, 128).half(), torch.randn(NB, 1, BS, 128, generator=g).half()
    kk[bt[0].long()[t // BS], 0, t % BS] = k.half()
    (kc, ks), (vc, vs) = F.encode(kk), F.encode(vv)
    return bt, [kc, vc, ks, vs], F.gather(vc, vs, bt[0], n)[0]


def _both(q, c, bt, n):
    """(decode, prefill) outputs of queries [T, G, 128] on one sequence's n keys, each query on all of them."""
    from microserve_b200 import kernels
    T = q.shape[0]
    many, lens = bt.expand(T, -1).contiguous().to(DEV), _i32([n] * T)
    d = _dev(c)
    return (kernels.paged_decode_fp4(q.to(DEV), *d, lens, many, SCALE).cpu().double(),
            kernels.paged_prefill_fp4(q.to(DEV), *d, many, _i32(range(T + 1)), lens, SCALE).cpu().double())


@pytest.mark.parametrize("n,G", [(1, 1), (64, 4), (65, 8), (700, 2), (2900, 7)])
def test_equal_scores_of_any_magnitude(n, G):
    """All keys alike, queries of 2^-4 to 2^15 of either sign: scores from 2^16 to 2^36 in the log2 domain and the
    same ones negative. Every product and sum is exact, so every weight is the same: the mean of the values."""
    bt, c, v = _filled(n, 64, torch.full((n, 128), 61440.0), 31)
    e = torch.arange(-4, 16)
    q = torch.cat([torch.exp2(e.double()), -torch.exp2(e.double())])[:, None, None].expand(-1, G, 128).half()
    mean, a = v.mean(0), v.abs().mean(0)
    decode, prefill = _both(q, c, bt, n)
    _within(decode, mean.expand_as(decode), a)
    _within(prefill, mean.expand_as(prefill), a, n, v.abs().max().item())


@pytest.mark.parametrize("n", [2, 150, 2000])
@pytest.mark.parametrize("sign", [1, -1])
def test_one_key_wins_by_far(n, sign):
    """Scores up to 2^35 in the log2 domain, one or two keys far above all others: their value, or the mean of two."""
    g = torch.Generator().manual_seed(n)
    for where in ({0}, {n - 1}, {n // 2}, {0, n - 1}, {n // 3, n // 2}):
        # positive queries: the winners are the largest; negative ones: the least negative
        k = (1000 * torch.rand(n, 128, generator=g) + 1) if sign > 0 else torch.full((n, 128), 60000.0)
        for w in where:
            k[w] = 60000.0 if sign > 0 else 30.0
        bt, c, v = _filled(n, 64, k, 32)
        q = torch.full((3, 4, 128), 60000.0 * sign).half()
        q[1] = 7.0 * sign
        q[2] = 900.0 * sign
        want, a = v[sorted(where)].mean(0), v[sorted(where)].abs().mean(0)
        decode, prefill = _both(q, c, bt, n)
        _within(decode, want.expand_as(decode), a)
        _within(prefill, want.expand_as(prefill), a, n, v.abs().max().item())


def _levels(lens, BS, Hkv, seed):
    """Keys of one element, of a few heights between 27648 and 38912, so that many are alike."""
    g = torch.Generator().manual_seed(seed)
    bt, NB = _tables(lens, BS, seed)
    k = torch.zeros(NB, Hkv, BS, 128, dtype=torch.float16)
    k[..., 0] = (28000 + 10000 * torch.rand(NB, Hkv, BS, generator=g)).half()
    v = torch.randn(NB, Hkv, BS, 128, generator=g).half()
    (kc, ks), (vc, vs) = F.encode(k), F.encode(v)
    return bt, [kc, vc, ks, vs]


def _expected(q, c, table, n, bad):
    """attend() of the oracle, with the pages `bad` masked."""
    Q, Hq, _ = q.shape
    BS, G = c[0].shape[2], Hq // c[0].shape[1]
    good = table.clone()
    good[good < 0] = 0
    k, v = F.gather(c[0], c[2], good, n), F.gather(c[1], c[3], good, n)
    t = torch.arange(n)
    seen = (t[None, :] <= (n - Q + torch.arange(Q))[:, None]) & ~torch.isin(t // BS, torch.tensor(bad))[None, :]
    o, a = torch.zeros(Q, Hq, 128, dtype=torch.float64), torch.zeros(Q, Hq, 128, dtype=torch.float64)
    for h in range(Hq):
        s = (q[:, h].double() @ k[h // G].t() * SCALE).masked_fill(~seen, float("-inf"))
        p = torch.softmax(s, -1).nan_to_num(0.0)  # a row that sees nothing
        o[:, h], a[:, h] = p @ v[h // G], p @ v[h // G].abs()
    return o, a


@pytest.mark.parametrize("Hq,Hkv,BS", [(16, 2, 64), (3, 1, 128), (8, 8, 64), (24, 4, 192)])
@pytest.mark.parametrize("masked", [False, True])
def test_far_and_near_rows_side_by_side(Hq, Hkv, BS, masked):
    """Rows with scores of 2^26 and more beside rows with scores of about 60, in items inside and across CTAs, with
    strided queries and, `masked`, pages outside the cache; far rows weigh the keys at the top level alike."""
    from microserve_b200 import _lib, kernels
    values = (2.0 ** 15, 2.0 ** -6, -(2.0 ** 15), 2.0 ** -7, 0.0, 2.0 ** 14, -(2.0 ** -6))
    seqs = [(70, 500), (3, 0), (0, 40), (129, 700), (1, 1800)]
    kv, cu = [q + p for q, p in seqs], [0]
    for n, _ in seqs:
        cu.append(cu[-1] + n)
    bt, c = _levels(kv, BS, Hkv, Hq)
    bad = {0: [1], 3: [0, 3], 4: [5]} if masked else {}
    for s, pages in bad.items():
        bt[s, pages] = torch.tensor([[-1, 1 << 30][i % 2] for i in range(len(pages))], dtype=torch.int32)
    tables = torch.where(bt >= c[0].shape[0], -1, bt)
    q = _one_element(cu[-1], Hq, values)
    wide = torch.full((cu[-1], Hq + 1, 128), 5.0, dtype=torch.float16)
    wide[:, :Hq] = q
    vmax = F.decode(c[1], c[3]).abs().max().item()
    want = [_expected(q[cu[s]:cu[s + 1]], c, tables[s], kv[s], bad.get(s, [])) for s in range(len(seqs)) if seqs[s][0]]
    o, a = torch.cat([x[0] for x in want]), torch.cat([x[1] for x in want])
    got = kernels.paged_prefill_fp4(wide.to(DEV)[:, :Hq], *_dev(c), bt.to(DEV), _i32(cu), _i32(kv), SCALE)
    _within(got, o, a, max(kv), vmax)
    # each sequence's last query, as a decode step
    last = [cu[s + 1] - 1 for s in range(len(seqs)) if seqs[s][0]]
    rows = [s for s in range(len(seqs)) if seqs[s][0]]
    got = kernels.paged_decode_fp4(wide[last].to(DEV)[:, :Hq], *_dev(c), _i32([kv[s] for s in rows]), bt[rows].to(DEV), SCALE)
    _within(got, o[last], a[last])
    assert _lib.device_status() == (3 if masked else 0)


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 1e8, 1e30, 2e38])
def test_softmax_scales_of_any_size(scale):
    """Scales so small that every key weighs the same and so large that scores times the scale pass fp32: the mean of
    all values, and of those of the largest score."""
    from microserve_b200 import kernels
    n, Hq, T = 900, 8, 40
    bt, c = _levels([n], 64, 2, 5)
    q = _one_element(T, Hq, (1.0, -1.0, 0.0, 2.0 ** 15, -64.0))
    o, a = F.attend(q, *c, bt[0], n, scale)
    vmax = F.decode(c[1], c[3]).abs().max().item()
    d = _dev(c)
    _within(kernels.paged_prefill_fp4(q.to(DEV), *d, bt.to(DEV), _i32([0, T]), _i32([n]), scale), o, a, n, vmax)
    got = kernels.paged_decode_fp4(q[-1:].to(DEV), *d, _i32([n]), bt.to(DEV), scale)
    _within(got, o[-1:], a[-1:])


def test_outputs_over_the_queries():
    """`out` is the query itself, or shares its memory: rows with far scores and without, items inside CTAs and across."""
    from microserve_b200 import kernels
    Hq, Hkv, seqs = 32, 8, [(64, 64)] * 60 + [(3, 1500)]
    kv, T = [a + b for a, b in seqs], sum(a for a, _ in seqs)
    bt, c = _levels(kv, 64, Hkv, 6)
    q = _one_element(T, Hq, (2.0 ** 15, 2.0 ** -6, -(2.0 ** 15), 0.0, 2.0 ** -7))
    cu = [64 * i for i in range(61)] + [T]
    args = (*_dev(c), bt.to(DEV), _i32(cu), _i32(kv), SCALE)
    want = kernels.paged_prefill_fp4(q.to(DEV), *args)
    same = q.to(DEV)
    assert kernels.paged_prefill_fp4(same, *args, out=same) is same and torch.equal(same, want)
    shared = torch.zeros(T + 3, Hq, 128, dtype=torch.float16, device=DEV)
    shared[3:] = q.to(DEV)
    got = kernels.paged_prefill_fp4(shared[3:], *args, out=shared[:T])
    assert torch.equal(got, want)
    last, args = q[-1:].to(DEV), (*_dev(c), _i32(kv[-1:]), bt[-1:].to(DEV), SCALE)
    want = kernels.paged_decode_fp4(last, *args)
    assert torch.equal(kernels.paged_decode_fp4(last, *args, out=last), want)
