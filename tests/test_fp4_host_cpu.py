"""The 4-bit cache's host side without a GPU: what the engine reserves for it, and calls
that are refused before any launch."""
from types import SimpleNamespace

import pytest
import torch

from microserve_b200 import kernels
from tests.test_fp4_cpu import INVALID, UNSUPPORTED, _decode, _prefill


@pytest.mark.parametrize("kind", ["fp8_e4m3", "fp4_e2m1"])
def test_the_fp8_attention_s_partials_are_reserved_for_the_fp8_cache_only(kind, monkeypatch):
    from microserve_b200.engine.model_runner import ModelRunner
    r = ModelRunner.__new__(ModelRunner)
    r.config = SimpleNamespace(kv_cache_dtype=kind)
    r.hf_config = SimpleNamespace(num_attention_heads=32)
    r.num_kv_heads, r.block_size, r.device, r.graph_bs = 8, 256, torch.device("cpu"), [1, 8]
    r.model = torch.nn.Module()
    asked = {}
    monkeypatch.setattr(kernels.workspace, "reserve", lambda n, device, name: asked.__setitem__(name, n))
    r._reserve_workspace(8, 16)
    assert (asked["decode"] > 0) == (kind == "fp8_e4m3") and asked["argmax"] > 0


@pytest.mark.parametrize("call", [_decode, _prefill])
@pytest.mark.parametrize("scale", [2.4e38, 3e38])
def test_scales_whose_log2_form_is_infinite_are_refused(call, scale):
    assert call(scale=scale) == INVALID


@pytest.mark.parametrize("B,Hq,Hkv,bs,mb", [
    (1 << 20, 16, 8, 256, 1 << 22),               # 2^30 tokens a row in 2^20 rows of 8 heads
    (65536, 64, 8, 512, 1 << 21), (1 << 30, 512, 512, 64, 1 << 24),
])
def test_decode_refuses_more_tiles_a_cta_than_32_bits_count(B, Hq, Hkv, bs, mb):
    assert _decode(qs=Hq * 128, B=B, Hq=Hq, Hkv=Hkv, bs=bs, mb=mb, wb=1 << 60) == UNSUPPORTED
