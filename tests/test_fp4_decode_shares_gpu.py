"""Decode attention over the 4-bit KV cache where shares begin and end inside, between and right behind items:
batches of one-tile sequences, of many lengths, and one long sequence among short ones."""
import random

import pytest
import torch

from oracle import fp4_kv as F
from tests.test_fp4_gpu import DEV, SCALE, _cache, _close, _dev, _i32, _status_clean, _tables  # noqa: F401

pytestmark = pytest.mark.gpu


def _lens(n, hi, seed, empty=0.1):
    r = random.Random(seed)
    return [0 if r.random() < empty else r.randint(1, hi) for _ in range(n)]


@pytest.mark.parametrize("lens,Hq,Hkv,BS", [
    ([32] * 300, 8, 8, 64), ([1] * 777, 2, 2, 64), ([33] * 150, 16, 4, 64), ([64] * 111, 8, 1, 128),
    (_lens(200, 400, 1), 32, 8, 256), (_lens(512, 70, 2, 0.5), 6, 1, 64), (_lens(40, 130, 3), 5, 1, 192),
    ([5000] + _lens(60, 90, 4), 16, 2, 256), (_lens(60, 90, 5) + [3001], 7, 1, 64), (_lens(9, 2000, 6), 24, 8, 256),
])
def test_shares_vs_oracle(lens, Hq, Hkv, BS):
    from microserve_b200 import kernels
    bt, NB = _tables(lens, BS, 11)
    c = _cache(NB, BS, Hkv, 12)
    q = torch.randn(len(lens), Hq, 128, generator=torch.Generator().manual_seed(13)).half()
    o, a = F.decode_attention(q, *c, lens, bt, SCALE)
    args = (q.to(DEV), *_dev(c), _i32(lens), bt.to(DEV), SCALE)
    first = kernels.paged_decode_fp4(*args)
    _close(first, o, a)
    for _ in range(20):  # the joins have one order: equal bits
        assert torch.equal(kernels.paged_decode_fp4(*args), first)
