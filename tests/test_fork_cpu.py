"""Forks of running sequences on the host: preemption among sequences that share their blocks, forks whose
page copies fail, forks in the middle of a prompt, and forks on two tensor-parallel ranks."""
import os
import random

import pytest
import torch.distributed as dist
import torch.multiprocessing as mp

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


def test_fork_in_the_middle_of_a_prompt():
    """22 tokens in chunks of 10: the fork shares the two full pages, gets a copy of the third and computes the rest
    of the prompt into pages of its own."""
    sched = Scheduler(16, 4, max_num_seqs=4, max_num_batched_tokens=10)
    seq = Sequence(list(range(22)), max_tokens=3)
    sched.add(seq)
    sched.postprocess(sched.schedule(), [None])
    assert seq.num_computed_tokens == 10
    child, copies = _fork(sched, seq)
    assert copies == [(seq.block_table[2], child.block_table[2], 2)] and child.block_table[:2] == seq.block_table[:2]
    assert child.gap == seq.gap == 12 and child.num_completion_tokens == 0
    while not sched.is_idle():
        batch = sched.schedule()
        sched.postprocess(batch, [7 if s.needs_sample else None for s in batch])
        if child.block_table and seq.block_table:
            assert not set(child.block_table[2:]) & set(seq.block_table[2:])
        _check_blocks(sched)
    assert seq.completion_token_ids == child.completion_token_ids == [7, 7, 7]
    assert sched.block_manager.free_blocks_nums == 16


class _Rank:
    """A tensor-parallel rank's runner without a GPU: records the page copies, and every rank gets rank 0's tokens."""

    def __init__(self):
        self.copies = []

    def copy_pages(self, pairs):
        self.copies.append(pairs)

    def execute(self, batch):
        tokens = [random.randrange(50) if s.needs_sample else None for s in batch]  # every rank its own, but for:
        dist.broadcast_object_list(tokens, src=0)
        return tokens


def _rank(rank, world, init_file, errq):
    try:
        dist.init_process_group("gloo", init_method=f"file://{init_file}", rank=rank, world_size=world)
        eng = LLMEngine.__new__(LLMEngine)
        eng.scheduler, eng.runner = Scheduler(20, 4, max_num_seqs=6, max_num_batched_tokens=12), _Rank()
        r = random.Random(5)  # the program, the same on every rank
        seqs = [eng.add(list(range(9 * i, 9 * i + 6 + 5 * i)), max_tokens=12) for i in range(3)]
        trace = []
        for step in range(200):
            if eng.is_idle():
                break
            if step % 3 == 1 and eng.scheduler.running:
                try:
                    seqs.append(eng.fork(r.choice(list(eng.scheduler.running))))
                except (RuntimeError, ValueError) as e:
                    trace.append(str(e))
            eng.step()
            base = seqs[0].seq_id
            trace.append([(s.seq_id - base, s.num_computed_tokens, list(s.block_table)) for s in eng.scheduler.running])
        trace += [eng.runner.copies, [s.token_ids for s in seqs]]
        assert eng.is_idle() and len(seqs) > 5 and eng.runner.copies
        both = [None] * world
        dist.all_gather_object(both, trace)
        assert both[0] == both[1]
        dist.barrier()
        dist.destroy_process_group()
    except Exception as ex:  # report to the parent
        import traceback
        errq.put(f"rank {rank}: {ex}\n{traceback.format_exc()}")
        raise
    os._exit(0)  # gloo's threads can abort a normal teardown


def test_forks_on_two_ranks_take_the_same_blocks(tmp_path):
    ctx = mp.get_context("spawn")
    errq = ctx.Queue()
    procs = [ctx.Process(target=_rank, args=(r, 2, str(tmp_path / "init"), errq)) for r in range(2)]
    for p in procs:
        p.start()
    for p in procs:
        p.join(180)
    alive = [p for p in procs if p.is_alive()]
    for p in alive:
        p.kill()
    assert not alive and all(p.exitcode == 0 for p in procs), errq.get() if not errq.empty() else "no answer"
