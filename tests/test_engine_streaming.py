"""Host side of long-running and branching sequences (CPU only): blocks freed
behind a sliding window, forks, packing the pool, sampling filters."""
import random

import pytest
import torch

from llm_from_scratch_amd.decode_model import DecodeModelConfig
from llm_from_scratch_amd.engine import BlockManager, SamplingParams, Scheduler, Sequence
from llm_from_scratch_amd.engine.block_manager import Block
from llm_from_scratch_amd.engine.llm_engine import check_window
from llm_from_scratch_amd.engine.model_runner import ModelRunner

BS = 16


@pytest.fixture(autouse=True)
def block_size_16():
    old = Sequence.block_size
    Sequence.block_size = BS
    yield
    Sequence.block_size = old


def consistent(bm, seqs):
    """Every block's count is its table entries', and used and free split the pool."""
    held = [b for s in seqs for b in s.block_table if b >= 0]
    assert {b: held.count(b) for b in set(held)} == {b: bm.blocks[b].ref_count for b in bm.used_block_ids}
    assert sorted(list(bm.used_block_ids) + list(bm.free_block_ids)) == list(range(len(bm.blocks)))
    assert all(bm.blocks[b].ref_count == 0 for b in bm.free_block_ids)


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (20, 4), (33, 17), (100, 1), (1000, 4)])
def test_blocks_behind_the_window_are_freed(window, sinks):
    """Exactly the blocks that no token from the newest on sees, but the last two."""
    bm = BlockManager(64, BS, window, sinks)
    s = Sequence(list(range(40)))
    bm.allocate(s)
    for step in range(300):
        s.append_token(step)
        bm.release_behind(s)
        assert bm.can_append(s)
        bm.append(s)
        p = s.num_tokens - 1
        for i, b in enumerate(s.block_table):
            rows = range(i * BS, (i + 1) * BS)
            seen = any(j < sinks or j > p - window for j in rows)
            assert (b >= 0) == (seen or i >= s.num_blocks - 2 or (i >= s.num_blocks - 3 and b >= 0)), (step, i)
        consistent(bm, [s])
    bm.deallocate(s)
    consistent(bm, [])
    assert s.num_released_blocks == 0


def test_a_sequence_may_outgrow_its_pool():
    bm = BlockManager(6, BS, window=32, sinks=4)
    s = Sequence(list(range(BS)))
    bm.allocate(s)
    for step in range(40 * BS):
        s.append_token(step % 7)
        bm.release_behind(s)
        assert bm.can_append(s)
        bm.append(s)
    assert s.num_blocks == 41 and len(bm.used_block_ids) <= 5


def test_release_leaves_shared_blocks_to_others():
    bm = BlockManager(32, BS, window=16, sinks=0)
    prompt = list(range(5 * BS + 3))
    a, b = Sequence(prompt), Sequence(prompt)
    bm.allocate(a)
    bm.allocate(b)
    assert b.num_cached_tokens == 5 * BS
    a.append_token(1)
    bm.release_behind(a)
    assert a.block_table[:4] == [-1] * 4 and a.block_table[4] >= 0
    consistent(bm, [a, b])
    assert all(x in bm.used_block_ids for x in b.block_table)


@pytest.mark.parametrize("n", [1, 15, 16, 17, 32, 47])
def test_fork_shares_full_blocks_and_copies_a_partial_one(n):
    """n tokens stored, one more sampled: the state between two steps."""
    sched = Scheduler(8, 1000, 32, BS, eos=-1)
    s = Sequence(list(range(n)), SamplingParams(top_k=3, top_p=0.5, max_tokens=99))
    sched.add_sequence(s)
    assert sched.schedule() == ([s], True)
    sched.postprocess([s], [7])
    (c, d), copies = sched.fork(s, 2)
    assert c.token_ids == s.token_ids and c.seq_id != s.seq_id != d.seq_id and c.seq_id != d.seq_id
    assert (c.top_k, c.top_p, c.max_tokens, c.num_prompt_tokens) == (3, 0.5, 99, n)
    if n % BS:
        assert copies == [(s.block_table[-1], c.block_table[-1]), (s.block_table[-1], d.block_table[-1])]
        assert len({s.block_table[-1], c.block_table[-1], d.block_table[-1]}) == 3
        assert c.block_table[:-1] == d.block_table[:-1] == s.block_table[:-1]
    else:
        assert copies == [] and c.block_table == d.block_table == s.block_table
    consistent(sched.block_manager, [s, c, d])
    # the branches go on by themselves
    for step in range(40):
        seqs, prefill = sched.schedule()
        assert not prefill and set(map(id, seqs)) == {id(s), id(c), id(d)}
        last = [x.block_table[-1] for x in seqs]
        assert len(set(last)) == 3
        sched.postprocess(seqs, [step, step + 100, step + 200])
        consistent(sched.block_manager, [s, c, d])
    assert s.token_ids[:n + 1] == c.token_ids[:n + 1] and s.token_ids[n + 1] != c.token_ids[n + 1]
    for x in (s, c, d):
        sched.block_manager.deallocate(x)
    consistent(sched.block_manager, [])


def test_fork_refusals():
    sched = Scheduler(8, 1000, 3, BS, eos=-1)
    s = Sequence(list(range(20)))
    with pytest.raises(ValueError, match="not running"):
        sched.fork(s)
    sched.add_sequence(s)
    sched.schedule()
    sched.postprocess([s], [1])
    with pytest.raises(RuntimeError, match="no free blocks"):
        sched.fork(s, 2)
    for n in (0, -1):
        with pytest.raises(ValueError, match="n must be"):
            sched.fork(s, n)
    assert len(sched.running) == 1
    consistent(sched.block_manager, [s])
    sched.fork(s, 1)


def test_pack_moves_the_used_blocks_down():
    rnd = random.Random(1)
    sched = Scheduler(64, 100000, 100, BS, eos=-1, sliding_window=40, num_sink_tokens=3)
    seqs = [Sequence([rnd.randrange(50) for _ in range(rnd.randrange(1, 90))]) for _ in range(12)]
    for s in seqs:
        sched.add_sequence(s)
    sched.schedule()
    sched.postprocess(seqs, [1] * len(seqs))
    sched.fork(seqs[0], 2)
    for s in seqs[::2]:  # holes
        sched.running.remove(s)
        sched.block_manager.deallocate(s)
    live = list(sched.running)
    bm = sched.block_manager
    content = {i: ("block", i) for i in range(100)}
    before = [[content[b] if b >= 0 else None for b in s.block_table] for s in live]
    hashes = {b: (bm.blocks[b].hash, bm.blocks[b].token_ids) for b in bm.used_block_ids}
    copies = sched.pack()
    assert copies and not set(s for s, _ in copies) & set(d for _, d in copies)
    for src, dst in copies:
        content[dst] = content[src]
    n = len(bm.used_block_ids)
    assert bm.used_block_ids == set(range(n))
    assert [[content[b] if b >= 0 else None for b in s.block_table] for s in live] == before
    for b in range(n):
        assert (bm.blocks[b].hash, bm.blocks[b].token_ids) == hashes[content[b][1]]
        if bm.blocks[b].hash != -1 and bm.hash_to_block_id[bm.blocks[b].hash] < n:
            assert bm.blocks[bm.hash_to_block_id[bm.blocks[b].hash]].hash == bm.blocks[b].hash
    consistent(bm, live)
    assert sched.pack() == []
    for _ in range(30):
        ran, _ = sched.schedule()
        sched.postprocess(ran, [2] * len(ran))
        consistent(bm, list(sched.running))


def test_a_shared_prefix_is_found_after_packing():
    bm = BlockManager(20, BS)
    gone, s = Sequence([9] * 40), Sequence(list(range(40)))
    bm.allocate(gone)
    bm.allocate(s)
    bm.deallocate(gone)
    copies = bm.pack()
    moved = dict(copies)
    s.block_table = [moved.get(b, b) for b in s.block_table]
    t = Sequence(list(range(40)))
    bm.allocate(t)
    assert t.num_cached_tokens == 32 and t.block_table[:2] == s.block_table[:2]
    consistent(bm, [s, t])


def test_preemption_spares_what_could_not_come_back():
    """Behind a window a sequence may be longer than the pool: another is
    preempted in its place, and without one the pool is too small."""
    sched = Scheduler(8, 1000, 5, BS, eos=-1, sliding_window=32)
    long = Sequence(list(range(10)), SamplingParams(max_tokens=10 ** 6))
    sched.add_sequence(long)
    for i in range(7 * BS):
        ran, _ = sched.schedule()
        assert ran == [long]
        sched.postprocess(ran, [i % 5])
    assert long.num_blocks > 5
    other = Sequence(list(range(8)), SamplingParams(max_tokens=10 ** 6))
    sched.add_sequence(other)
    preempted = 0
    for i in range(6 * BS):
        ran, _ = sched.schedule()
        assert ran
        assert long in sched.running
        preempted += other in sched.waiting
        sched.postprocess(ran, [3] * len(ran))
    consistent(sched.block_manager, [s for s in sched.running])
    alone = Scheduler(8, 1000, 3, BS, eos=-1, sliding_window=40)
    s = Sequence(list(range(10)), SamplingParams(max_tokens=10 ** 6))
    alone.add_sequence(s)
    with pytest.raises(RuntimeError, match="KV pool is full"):
        for i in range(10 * BS):
            ran, _ = alone.schedule()
            alone.postprocess(ran, [i % 5])


def test_the_same_tokens_behind_another_prefix_are_no_hit():
    """A block freed with its hash still known, then filled with the same tokens
    behind other ones: the first prompt must not find it."""
    p1, p2, x = list(range(BS)), list(range(100, 100 + BS)), list(range(50, 50 + BS))
    bm = BlockManager(5, BS)
    keep, a = Sequence(p1 + [7]), Sequence(p1 + x + [7])
    bm.allocate(keep)
    bm.allocate(a)
    block = a.block_table[1]
    bm.deallocate(a)
    spare = Sequence([1])  # frees leave the queue's front: block is next but one
    bm.allocate(spare)
    while bm.free_block_ids[1] != block:
        bm.free_block_ids.rotate(1)
    b = Sequence(p2 + x)  # its last block takes x after p2
    bm.allocate(b)
    assert b.block_table[1] == block
    bm.deallocate(spare)
    bm.free_block_ids.append(len(bm.blocks))
    bm.blocks.append(Block(len(bm.blocks)))
    c = Sequence(p1 + x + [7])
    bm.allocate(c)
    assert c.block_table[0] == keep.block_table[0] and c.block_table[1] != block and c.num_cached_tokens == BS


def test_packing_leaves_no_false_prefix():
    """The same where packing moves a block onto a freed one's place."""
    p1, p2, x = list(range(BS)), list(range(100, 100 + BS)), list(range(50, 50 + BS))
    bm = BlockManager(12, BS)
    keep, a, b = Sequence(p1 + [7]), Sequence(p1 + x + [7]), Sequence(p2 + x + [7])
    for s in (keep, a, b):
        bm.allocate(s)
    hole = a.block_table[1]
    bm.deallocate(a)
    moved = dict(bm.pack())
    b.block_table = [moved.get(i, i) for i in b.block_table]
    c = Sequence(p1 + x + [7])
    bm.allocate(c)
    assert hole in moved.values()
    assert c.block_table[0] == keep.block_table[0] and c.block_table[1] not in b.block_table
    assert c.num_cached_tokens == BS


def test_engine_and_model_windows_agree():
    class Layer(torch.nn.Module):
        def __init__(self, window, sinks):
            super().__init__()
            self.k_cache = self.v_cache = torch.empty(0)
            self.window, self.sinks = window, sinks

    model = torch.nn.Sequential(Layer(64, 4), Layer(32, 0))
    check_window(model, None, 0)
    check_window(model, 64, 4)
    check_window(model, 100, 16)
    for window, sinks in ((63, 4), (64, 3)):
        with pytest.raises(ValueError, match="the engine keeps"):
            check_window(model, window, sinks)
    with pytest.raises(ValueError, match="window of None"):
        check_window(torch.nn.Sequential(Layer(None, 0)), 64, 4)


def test_sampling_params_and_filters():
    for bad in (dict(top_k=-1), dict(top_k=2 ** 31), dict(top_p=0.0), dict(top_p=1.1), dict(min_p=-0.1), dict(min_p=2.0)):
        with pytest.raises(AssertionError):
            SamplingParams(**bad)
    runner = ModelRunner.__new__(ModelRunner)
    assert ModelRunner.prepare_filters(runner, [Sequence([1]), Sequence([2], SamplingParams(temperature=0.5))]) == {}


def test_config_refusals():
    with pytest.raises(ValueError, match="qk_norm"):
        DecodeModelConfig(qk_norm="heads")
    with pytest.raises(ValueError, match="window"):
        DecodeModelConfig(sliding_window=0)
    with pytest.raises(ValueError, match="sinks"):
        DecodeModelConfig(num_sink_tokens=4)
    cfg = DecodeModelConfig(sliding_window=128, num_sink_tokens=4, qk_norm="head")
    rc = cfg.runner_config()
    assert rc["sliding_window"] == 128 and rc["num_sink_tokens"] == 4
    assert cfg.reference_state_keys()["layers.0.att.q_norm.weight"] == (64,)
    assert DecodeModelConfig().reference_state_keys()["layers.0.att.q_norm.weight"] == (768,)
