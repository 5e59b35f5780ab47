"""Reading the 4-bit KV cache on both sides of the number of rows from which a lane takes two tokens, odd token
counts among them."""
import pytest
import torch

from oracle import fp4_kv as F
from tests.test_fp4_gpu import DEV, _cache, _dev, _status_clean  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,more", [(8, -1), (8, 0), (8, 1), (1, 0), (1, 5), (3, 16), (5, -1)])
def test_load_bit_exact_around_the_two_token_rule(H, more):
    from microserve_b200 import kernels
    sms = torch.cuda.get_device_properties(DEV).multi_processor_count
    T = (sms * 8 * 16 + H - 1) // H + more
    BS, NB = 256, 4
    c = _cache(NB, BS, H, H)
    slots = torch.randint(-1, NB * BS, (T,), generator=torch.Generator().manual_seed(T))
    s = slots.clamp_min(0)
    for got, codes, scales in zip(kernels.load_kv_fp4(*_dev(c), slots.to(DEV)), c[:2], c[2:]):
        ref = F.decode(codes[s // BS, :, s % BS], scales[s // BS, :, s % BS])
        assert torch.equal(got.cpu().double(), torch.where((slots >= 0)[:, None, None], ref, torch.zeros_like(ref)))
