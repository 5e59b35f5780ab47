"""The 4-bit cache's host side without a GPU: what the engine reserves for it, and calls
that are refused before any launch."""
from types import SimpleNamespace

import pytest
import torch

from microserve_b200 import kernels
from tests.test_fp4_cpu import INVALID, _decode, _prefill


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
