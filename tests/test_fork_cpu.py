"""Forks of running sequences on the host: preemption among sequences that share their blocks, and forks whose
page copies fail."""
import random

import pytest

from microserve_b200.engine.llm import LLMEngine
from microserve_b200.engine.scheduler import Scheduler
from microserve_b200.engine.sequence import Sequence, SequenceStatus
from tests.test_fp4_cpu import _fork, _running


def _prompts(blocks, *lens, **kw):
    """A scheduler whose first step ran prompts of these lengths (pages of 4 tokens)."""
    sched = Scheduler(blocks, 4, max_num_seqs=8, **kw)
    seqs = [Sequence([100 * i + t for t in range(n)], max_tokens=64) for i, n in enumerate(lens)]
    for s in seqs:
        sched.add(s)
    sched.postprocess(sched.schedule(), [7] * len(seqs))
    return sched, *seqs


def _check_blocks(sched):
    """Reference counts and the free and used blocks agree with the running sequences' tables."""
    bm = sched.block_manager
    refs = [0] * len(bm.blocks)
    for seq in sched.running:
        for b in seq.block_table:
            refs[b] += 1
    assert [b.ref_count for b in bm.blocks] == refs
    assert bm.used_blocks == {i for i, n in enumerate(refs) if n} and len(bm.free_blocks) == refs.count(0)
    assert all(not s.block_table for s in sched.waiting)


def test_a_step_is_scheduled_though_the_newest_victim_frees_nothing():
    """8 and 5 tokens fill four pages; a fork of the first, at its page border, owns none of its own."""
    sched, seq, other = _prompts(4, 8, 5)
    child, copies = _fork(sched, seq)
    assert copies == [] and sched.block_manager.free_blocks_nums == 0
    batch = sched.schedule()
    # both need a page; the one sequence that has some to give is the other one, and the fork keeps its progress
    assert batch == [seq, child] and list(sched.waiting) == [other]
    sched.postprocess(batch, [1, 2])
    _check_blocks(sched)


def test_victims_are_taken_until_a_block_is_free():
    """Two forks share all their pages with one another only: neither frees one alone, both together do."""
    sched, needs, parent = _prompts(5, 8, 12)
    forks = [_fork(sched, parent)[0] for _ in range(2)]
    sched._retire(parent)
    assert sched.block_manager.free_blocks_nums == 0
    batch = sched.schedule()
    assert batch == [needs] and len(needs.block_table) == 3 and list(sched.waiting) == forks
    sched.postprocess(batch, [1])
    _check_blocks(sched)


@pytest.mark.parametrize("seed", range(60))
def test_forked_runs_come_to_an_end(seed):
    """Random forks in a cache that is too small for all of them: no step is empty before everything has finished,
    and every sequence gets all its tokens."""
    r = random.Random(seed)
    sched = Scheduler(r.randint(10, 14), 4, max_num_seqs=r.randint(3, 8), max_num_batched_tokens=r.choice((8, 64)))
    seqs = [_running(sched, r.randint(2, 16), max_tokens=r.randint(2, 16)) for _ in range(3)]
    for _ in range(3000):
        if sched.is_idle():
            break
        if r.random() < 0.3 and sched.running and len(seqs) < 12:
            try:
                seqs.append(_fork(sched, r.choice(list(sched.running)))[0])
            except (RuntimeError, ValueError):
                pass
        batch = sched.schedule()
        assert batch, "a step without work"
        sched.postprocess(batch, [r.randint(0, 3) if s.needs_sample else None for s in batch])
        _check_blocks(sched)
    assert sched.is_idle() and all(s.status == SequenceStatus.FINISHED for s in seqs)
    assert all(s.num_completion_tokens == s.max_tokens for s in seqs)
    assert not sched.block_manager.used_blocks


class _NoCopies:
    def copy_pages(self, pairs):
        raise MemoryError("no room for the copies' arguments")


def test_a_fork_whose_copies_fail_leaves_nothing_behind():
    sched, seq = _prompts(6, 10)
    eng = LLMEngine.__new__(LLMEngine)
    eng.scheduler, eng.runner = sched, _NoCopies()
    bm = sched.block_manager
    cached = dict(bm.hash_to_block)
    with pytest.raises(MemoryError):
        eng.fork(seq)
    assert list(sched.running) == [seq] and not sched.waiting
    assert bm.free_blocks_nums == 3 and bm.hash_to_block == cached
    _check_blocks(sched)
    for _ in range(8):  # `seq` goes on alone
        assert sched.schedule() == [seq]
        sched.postprocess([seq], [3])
        _check_blocks(sched)
