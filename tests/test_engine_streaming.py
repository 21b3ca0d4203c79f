"""Host side of long-running and branching sequences (CPU only): blocks freed
behind a sliding window, forks, packing the pool, sampling filters."""
import random

import pytest
import torch

from llm_from_scratch_amd.decode_model import DecodeModelConfig
from llm_from_scratch_amd.engine import BlockManager, SamplingParams, Scheduler, Sequence
from llm_from_scratch_amd.engine.block_manager import Block
from llm_from_scratch_amd.engine.llm_engine import check_window
from llm_from_scratch_amd.engine.model_runner import ModelRunner, prefill_metadata, prefill_parts

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


def in_one_queue(sched, seqs):
    """Every sequence is finished or in one queue once, and the blocks held are the running ones'."""
    for s in seqs:
        assert s.is_finished + sched.waiting.count(s) + sched.running.count(s) == 1, s.seq_id
    consistent(sched.block_manager, list(sched.running))


def drive(sched, seqs, steps=20000):
    """Run to the end, the queues looked at after every step."""
    for i in range(steps):
        if sched.is_finished():
            break
        ran, _ = sched.schedule()
        in_one_queue(sched, seqs)
        sched.postprocess(ran, [i % 7] * len(ran))
    assert all(s.is_finished for s in seqs)
    assert not sched.block_manager.used_block_ids


def test_a_sequence_past_the_pool_waits_for_one_that_runs_on():
    """The last running sequence needs a block, is longer than the pool and so
    cannot be preempted, but one before it goes on: it waits for its blocks."""
    sched = Scheduler(8, 1000, 6, BS, eos=-1, sliding_window=48)
    seqs = [Sequence([i] * n, SamplingParams(max_tokens=m)) for i, (n, m) in
            enumerate([(7, 60), (71, 70), (53, 20), (54, 20)])]
    for s in seqs:
        sched.add_sequence(s)
    drive(sched, seqs)
    # a stream past its pool and its fork
    sched = Scheduler(8, 1000, 5, BS, eos=-1, sliding_window=2 * BS)
    stream = Sequence([1] * 10, SamplingParams(max_tokens=12 * BS))
    sched.add_sequence(stream)
    for i in range(8 * BS):
        ran, _ = sched.schedule()
        sched.postprocess(ran, [i % 5])
    assert stream.num_blocks > 5
    children, _ = sched.fork(stream, 1)
    drive(sched, [stream, *children])


def test_the_queues_stand_when_the_pool_is_too_small():
    """Two sequences longer than the pool, both without a block to go on with:
    the error takes neither out of its queue."""
    sched = Scheduler(8, 1000, 4, BS, eos=-1, sliding_window=40)
    stream = Sequence([1] * 10, SamplingParams(max_tokens=10 ** 6))
    sched.add_sequence(stream)
    while stream.num_tokens % BS or stream.num_blocks <= 5:
        ran, _ = sched.schedule()
        sched.postprocess(ran, [3] * len(ran))
    seqs = [stream, *sched.fork(stream, 1)[0]]
    held = None
    for i in range(20 * BS):
        try:
            ran, _ = sched.schedule()
        except RuntimeError as e:
            assert "KV pool is full" in str(e)
            held = [list(s.block_table) for s in seqs]
            break
        in_one_queue(sched, seqs)
        sched.postprocess(ran, [3] * len(ran))
    assert held is not None and list(sched.running) == seqs
    in_one_queue(sched, seqs)
    with pytest.raises(RuntimeError, match="KV pool is full"):  # again, with everything as it was
        sched.schedule()
    assert [s.block_table for s in seqs] == held and list(sched.running) == seqs
    # one of them given up, the other goes on
    sched.running.remove(seqs[0])
    sched.block_manager.deallocate(seqs[0])
    assert sched.schedule() == ([seqs[1]], False)


@pytest.mark.parametrize("budget", [10 ** 6, 128, 40])
def test_streams_of_any_lengths_finish_or_the_pool_is_full(budget):
    """Random lengths, windows, pools and forks: every sequence finishes, or no
    running one fits the pool or has a block to go on with."""
    rnd = random.Random(budget)
    ended = 0
    for case in range(150):
        pool, window = rnd.randrange(3, 12), rnd.choice([None, 1, BS, 32, 48, 100])
        sched = Scheduler(rnd.randrange(1, 6), budget, pool, BS, eos=-1, sliding_window=window, num_sink_tokens=0 if window is None else rnd.choice([0, 4]))
        longest = min(budget, (pool - 1) * BS)
        seqs = [Sequence([rnd.randrange(3)] * rnd.randrange(1, longest), SamplingParams(max_tokens=rnd.randrange(1, 9 * BS)))
                for _ in range(rnd.randrange(1, 6))]
        for s in seqs:
            sched.add_sequence(s)
        for step in range(20000):
            if sched.is_finished():
                break
            try:
                ran, _ = sched.schedule()
            except RuntimeError:
                in_one_queue(sched, seqs)
                assert sched.running and not sched.block_manager.free_block_ids
                assert all(s.num_blocks > pool and s.num_tokens % BS == 1 for s in sched.running)
                break
            in_one_queue(sched, seqs)
            sched.postprocess(ran, [step % 5] * len(ran))
            if sched.running and rnd.random() < 0.01 and sched.block_manager.can_fork(sched.running[0]):
                seqs += sched.fork(sched.running[0])[0]
        else:
            raise AssertionError("no end")
        ended += sched.is_finished()
    assert ended > 75


def test_a_sequence_past_the_token_budget_is_resumed():
    """Preempted with more tokens than a prefill takes, it comes back alone,
    and those behind it after it; a fresh prompt past the budget still waits."""
    sched = Scheduler(8, 128, 10, BS, eos=-1, sliding_window=32)
    seqs = [Sequence([i] * n, SamplingParams(max_tokens=60)) for i, n in enumerate([111, 15, 33, 123])]
    for s in seqs:
        sched.add_sequence(s)
    drive(sched, seqs)
    sched = Scheduler(8, 128, 20, BS, eos=-1)
    old, other, fresh = Sequence([1] * 120, SamplingParams(max_tokens=60)), Sequence([2] * 9), Sequence([3] * 129)
    sched.add_sequence(old)
    for _ in range(30):
        ran, _ = sched.schedule()
        sched.postprocess(ran, [5])
    sched.running.remove(old)
    sched.preempt(old)
    sched.add_sequence(other)
    sched.add_sequence(fresh)
    assert old.num_tokens == 150 and sched.schedule() == ([old], True)
    sched.postprocess([old], [5])
    assert sched.schedule() == ([other], True)
    sched.postprocess([other], [5])
    ran, prefill = sched.schedule()
    assert ran == [old, other] and not prefill and list(sched.waiting) == [fresh]


@pytest.mark.parametrize("budget", [1, 16, 40, 64, 1000])
@pytest.mark.parametrize("n,shared", [(33, 0), (200, 0), (208, 0), (209, 96)])
def test_parts_of_a_resumed_prefill(budget, n, shared):
    """The parts together are the whole prefill: its tokens, positions and
    slots, each behind those before it, whole blocks within the budget."""
    bm = BlockManager(64, BS)
    prompt = [i % 91 for i in range(n)]
    other = Sequence(prompt[:shared] + [5])
    bm.allocate(other)
    s = Sequence(prompt[:20])
    for t in prompt[20:]:
        s.append_token(t)
    bm.allocate(s)
    assert s.num_cached_tokens == shared
    parts = prefill_parts([s], BS, budget)
    whole = prefill_metadata([s], BS)
    each = [prefill_metadata(p, BS) for p in parts]
    for key in ("input_ids", "positions", "slot_mapping"):
        assert sum((m[key] for m in each), []) == whole[key]
    at = shared
    for i, m in enumerate(each):
        size = len(m["input_ids"])
        assert size <= max(budget, BS) and (size % BS == 0 or i == len(each) - 1)
        at += size
        assert m["cu_seqlens_q"] == [0, size] and m["cu_seqlens_k"] == [0, at]
        assert parts[i][0].block_table == s.block_table[:-(-at // BS)]
    assert s.num_tokens == n and len(s.block_table) == s.num_blocks  # as it was
    fresh = Sequence(prompt)
    assert prefill_parts([fresh], BS, budget) == [[fresh]] and prefill_parts([s, fresh], BS, budget) == [[s, fresh]]


def test_a_layer_that_knows_no_window_is_refused():
    """Layers that the runner gives a pool are those whose blocks are freed: one
    without a window of its own sees everything."""
    class Plain(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.k_cache = self.v_cache = torch.empty(0)

    class Windowed(Plain):
        window, sinks = 64, 4

    class NoSinks(Plain):
        window = 64

    class Projection(torch.nn.Module):  # no pool: not asked
        window = None

    model = torch.nn.Sequential(Projection(), Windowed(), Plain())
    check_window(model, None, 0)
    with pytest.raises(ValueError, match="2 sees a window of None"):
        check_window(model, 64, 4)
    check_window(torch.nn.Sequential(Projection(), Windowed(), NoSinks()), 64, 4)
    for bad in ((0, 0), (-1, 0), (64, -1)):
        with pytest.raises(ValueError, match="window must be >= 1"):
            check_window(torch.nn.Sequential(), *bad)
