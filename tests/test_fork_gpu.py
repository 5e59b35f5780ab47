"""LLMEngine.fork in the middle of a chunked prompt, on both caches."""
import pytest
import torch

from tests.test_fp4_gpu import _engine, _status_clean  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["fp8_e4m3", "fp4_e2m1"])
def test_fork_in_the_middle_of_a_prompt(kind):
    """The prompt takes three steps; the fork comes after the second. Its pages hold what the parent's do up to
    there, in every layer, and both sequences go through the rest and their tokens, each in its own pages."""
    from microserve_b200.engine.sequence import SamplingParams
    prompt = torch.randint(100, 4096, (500,), generator=torch.Generator().manual_seed(3)).tolist()
    eng = _engine(kind, True)
    seq = eng.add(prompt, SamplingParams(temperature=0.0), max_tokens=6)
    for _ in range(2):
        eng.step()
    assert seq.num_computed_tokens == 400 and seq.num_completion_tokens == 0
    child = eng.fork(seq)
    assert child.block_table[0] == seq.block_table[0] and child.block_table[1] != seq.block_table[1]
    at = 3 if kind == "fp8_e4m3" else 4
    codes, scales = eng.runner.kv_cache.view(torch.uint8), eng.runner.kv_scale_cache
    pages = [t.narrow(at, 0, 400 - 256) for t in (codes, scales)]
    for t in pages:
        mine, its = t[:, :, child.block_table[1]], t[:, :, seq.block_table[1]]
        assert torch.equal(mine, its) and (mine != 0).any()
    while not eng.is_idle():
        eng.step()
    assert len(seq.completion_token_ids) == len(child.completion_token_ids) == 6
    assert child.token_ids[:500] == prompt and child.num_prompt_tokens == 500
    assert eng.scheduler.block_manager.free_blocks_nums == 12
