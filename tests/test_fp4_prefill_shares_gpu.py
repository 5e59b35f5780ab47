"""Chunk-prefill attention over the 4-bit KV cache where its list of steps is dealt to many CTAs: items that
cross CTAs, CTAs with many items, tiles without rows among full ones, and Q rows that other sequences own."""
import random

import pytest
import torch

from oracle import fp4_kv as F
from tests.test_fp4_gpu import DEV, SCALE, _cache, _close, _dev, _i32, _status_clean, _tables  # noqa: F401

pytestmark = pytest.mark.gpu


def _inputs(seqs, Hq, Hkv, BS, seed=3):
    kv = [q + p for q, p in seqs]
    bt, NB = _tables(kv, BS, seed)
    cu = [0]
    for n, _ in seqs:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1], Hq, 128, generator=torch.Generator().manual_seed(seed)).half()
    return q, _cache(NB, BS, Hkv, seed), bt, cu, kv


def _check(seqs, Hq, Hkv, BS, runs=1):
    from microserve_b200 import kernels
    q, c, bt, cu, kv = _inputs(seqs, Hq, Hkv, BS)
    o, a = F.prefill_attention(q, *c, bt, cu, kv, SCALE)
    args = (q.to(DEV), *_dev(c), bt.to(DEV), _i32(cu), _i32(kv), SCALE)
    first = kernels.paged_prefill_fp4(*args)
    _close(first, o, a, prefill=True)
    for _ in range(runs - 1):  # the joins have one order: equal bits
        assert torch.equal(kernels.paged_prefill_fp4(*args), first)


def _many(n, qhi, phi, seed):
    r = random.Random(seed)
    return [(r.choice((0, 1, r.randint(1, qhi))), r.randint(0, phi)) for _ in range(n)]


@pytest.mark.parametrize("seqs,Hq,Hkv,BS", [
    (_many(33, 60, 200, 1), 16, 2, 64),     # more sequences than a warp has lanes
    (_many(64, 9, 90, 2), 8, 8, 128),
    (_many(150, 3, 130, 3), 3, 1, 64),      # G = 3: 126 rows a tile
    (_many(600, 2, 70, 4), 16, 2, 64),      # a CTA has many items of a step or two
    ([(1, 20000)], 8, 1, 256),              # one item over all CTAs
    ([(2, 9000), (1, 3), (65, 6000)], 14, 2, 192),
    ([(1000, 0)], 16, 2, 64),               # items of 1 to 16 steps
    ([(33, 500), (16, 500), (32, 500), (17, 500)] * 6, 16, 2, 128),  # second tiles with 1, 0, 16, 1 tokens
])
def test_shares_vs_oracle(seqs, Hq, Hkv, BS):
    _check(seqs, Hq, Hkv, BS, runs=3)


def test_runs_are_equal():
    """Mixed items many times over: a step out of order would show as a difference."""
    _check([(33, 900), (16, 40), (200, 300), (1, 1500), (5, 0), (129, 64)], 24, 4, 64, runs=200)


@pytest.mark.parametrize("Hq,Hkv", [(16, 2), (3, 1), (8, 8)])
def test_nan_in_an_item_over_many_ctas(Hq, Hkv):
    """A NaN of V late in a long item reaches the rows that see it, in its 16 columns, and nothing else."""
    from microserve_b200 import kernels
    BS, n = 64, 3000
    q, c, bt, cu, kv = _inputs([(40, n - 40), (7, 100)], Hq, Hkv, BS)
    at = n - 20  # position of the NaN: seen by the last 20 queries
    o, a = F.prefill_attention(q, *c, bt, cu, kv, SCALE)  # without it, for all that it leaves alone
    c[3][int(bt[0, at // BS]), Hkv - 1, at % BS, 5] = 255
    got = kernels.paged_prefill_fp4(q.to(DEV), *_dev(c), bt.to(DEV), _i32(cu), _i32(kv), SCALE)
    want = torch.zeros(got.shape, dtype=torch.bool)
    want[20:40, -(Hq // Hkv):, 80:96] = True
    assert torch.equal(torch.isnan(got).cpu(), want)
    _close(torch.where(want, 0, got.cpu()), torch.where(want, 0, o), torch.where(want, 0, a), prefill=True)


@pytest.mark.parametrize("Hq,Hkv,lead", [(6, 2, 8), (8, 1, 0), (7, 7, 24)])
def test_strided_queries_and_rows_of_others(Hq, Hkv, lead):
    """Queries inside wider rows; NaN and infinite queries of the other sequences, and of the elements between the
    rows, stay out of a sequence's rows."""
    from microserve_b200 import kernels
    BS = 64
    q, c, bt, cu, kv = _inputs([(3, 70), (5, 0), (90, 33)], Hq, Hkv, BS)
    q[3] = float("nan")
    q[5] = float("inf")
    wide = torch.full((cu[-1], Hq * 128 + 64), float("nan"), dtype=torch.float16)
    view = wide[:, lead:lead + Hq * 128].view(cu[-1], Hq, 128)
    view.copy_(q)
    dev = wide.to(DEV)[:, lead:lead + Hq * 128].view(cu[-1], Hq, 128)
    assert not dev.is_contiguous()
    got = kernels.paged_prefill_fp4(dev, *_dev(c), bt.to(DEV), _i32(cu), _i32(kv), SCALE).cpu()
    keep = [i for i in range(cu[-1]) if i not in (3, 5)]
    o, a = F.prefill_attention(torch.where(torch.isfinite(q), q, 0), *c, bt, cu, kv, SCALE)
    _close(got[keep], o[keep], a[keep], prefill=True)


def test_starts_outside_the_queries():
    """Starts past the queries or in falling order leave out rows, and no row behind the queries is touched."""
    from microserve_b200 import kernels
    q, c, bt, cu, kv = _inputs([(30, 50), (20, 80), (10, 0)], 8, 2, 64)
    args = (q.to(DEV), *_dev(c), bt.to(DEV))
    want = kernels.paged_prefill_fp4(*args, _i32(cu), _i32(kv), SCALE)
    out = torch.full((60, 8, 128), 3.25, dtype=torch.float16, device=DEV)
    kernels.paged_prefill_fp4(*args, _i32([0, 30, 25, 1 << 30]), _i32([80, 100, 35]), SCALE, out=out)
    assert torch.equal(out[:25], want[:25])
    assert torch.isfinite(out).all()


def test_two_calls_at_once():
    """The same and other batches on two streams at once, each many times: a call has its own workspace."""
    from microserve_b200 import kernels
    sets = []
    for seed, seqs in ((5, [(60, 2000), (9, 100)]), (6, [(300, 300)])):
        q, c, bt, cu, kv = _inputs(seqs, 16, 4, 64, seed)
        args = (q.to(DEV), *_dev(c), bt.to(DEV), _i32(cu), _i32(kv), SCALE)
        sets.append((args, kernels.paged_prefill_fp4(*args)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(40):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                args, want = sets[(i + k) % 2]
                got.append((kernels.paged_prefill_fp4(*args), want))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for g, w in got)
