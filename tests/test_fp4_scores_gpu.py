"""The attentions over the 4-bit KV cache where scores climb, fall and jump along a sequence, so that the softmax
reference moves and what was summed is rescaled.

Only element 0 of the queries and keys is not zero, and it has few bits, so a score is exact in
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
