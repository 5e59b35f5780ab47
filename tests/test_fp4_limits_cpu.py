"""Limits of the operators on the 4-bit cache that hold before any launch."""
import pytest

from microserve_b200 import _lib
from tests.test_fp4_cpu import UNSUPPORTED, _prefill


@pytest.mark.parametrize("n,T,Hq,Hkv,mb", [
    (1 << 20, 1 << 20, 8, 8, 1 << 16),          # sequences x pages
    (1, (1 << 31) - 1, 64, 8, 1 << 20),         # tokens x pages
    (40000, 40000, 256, 256, 512),              # heads
])
def test_prefill_refuses_more_steps_than_32_bits_count(n, T, Hq, Hkv, mb):
    assert _prefill(qs=Hq * 128, n=n, T=T, Hq=Hq, Hkv=Hkv, mb=mb) == UNSUPPORTED
    assert b"unsupported" in _lib.load().ms_last_error()
