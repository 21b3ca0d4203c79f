"""Prefill-first scheduler with preemption, as engine/scheduler.py of the
reference (same queues, policy and stopping rules).

Behavioural fixes (the reference's bugs are not copied):
  * a running sequence popped when the decode batch is already full goes
    back to the front of ``running`` (the reference's ``break`` at :59-61
    drops it from every queue);
  * after preempting the newest running sequence the current one is retried
    with the freed blocks (the reference, :53-54, drops it);
  * ``max_tokens`` stops a sequence after exactly ``max_tokens`` completion
    tokens (the reference's ``1 + num_completion_tokens`` test, :89, stops
    one token early);
  * a preempted sequence that grew past ``max_num_batched_tokens`` is
    resumed (asked for its whole length within the budget, it would wait at
    the queue's head for good).
"""
from __future__ import annotations

from collections import deque
from typing import Optional

from .block_manager import BlockManager
from .sequence import Sequence, SequenceStatus


class Scheduler:
    def __init__(self, max_num_sequences: int, max_num_batched_tokens: int, max_cached_blocks: int,
                 block_size: int, eos: int, sliding_window: Optional[int] = None, num_sink_tokens: int = 0):
        self.block_manager = BlockManager(max_cached_blocks, block_size, sliding_window, num_sink_tokens)
        self.max_num_batched_tokens = max_num_batched_tokens
        self.max_num_sequences = max_num_sequences
        self.waiting: deque[Sequence] = deque()
        self.running: deque[Sequence] = deque()
        self.eos = eos

    def is_finished(self) -> bool:
        return not self.waiting and not self.running

    def add_sequence(self, sequence: Sequence) -> None:
        self.waiting.append(sequence)

    def schedule(self) -> tuple[list[Sequence], bool]:
        """Prefill as many waiting sequences as fit; otherwise one decode token
        for each running sequence, preempting the newest ones when the pool
        cannot hold another block (engine/scheduler.py:26-69)."""
        scheduled: list[Sequence] = []
        num_tokens = 0
        while self.waiting and len(scheduled) < self.max_num_sequences:
            seq = self.waiting[0]
            # a preempted sequence that outgrew the budget while decoding comes
            # back alone (the runner prefills it in parts)
            outgrew = not scheduled and seq.num_completion_tokens > 0
            if (self.block_manager.can_allocate(seq)
                    and (len(seq) + num_tokens <= self.max_num_batched_tokens or outgrew)):
                self.waiting.popleft()
                self.block_manager.allocate(seq)
                seq.status = SequenceStatus.RUNNING
                self.running.append(seq)
                scheduled.append(seq)
                num_tokens += len(seq)
            else:
                break
        if scheduled:
            return scheduled, True

        order = list(self.running)
        stalled = False
        while self.running:
            seq = self.running.popleft()
            self.block_manager.release_behind(seq)
            if not self.block_manager.can_append(seq):
                victim = self._victim([seq, *self.running])
                if victim is None:  # seq waits for the blocks of those that go on
                    stalled = True
                    continue
                if victim is not seq:  # seq is tried again with the freed blocks
                    self.running.remove(victim)
                    self.running.appendleft(seq)
                self.preempt(victim)
                continue
            if num_tokens >= self.max_num_batched_tokens or len(scheduled) >= self.max_num_sequences:
                break
            self.block_manager.append(seq)
            scheduled.append(seq)
            num_tokens += 1
        self.running = deque(s for s in order if s.status == SequenceStatus.RUNNING)
        if stalled and not scheduled:
            raise RuntimeError("the KV pool is full, and no running sequence fits it to be resumed later")
        return scheduled, False

    def _victim(self, among: list[Sequence]) -> Optional[Sequence]:
        """The newest sequence whose context the pool can hold at once, as its
        prefill will ask: behind a sliding window one may outgrow the pool, and
        could never be resumed."""
        total = len(self.block_manager.blocks)
        return next((seq for seq in reversed(among) if seq.num_blocks <= total), None)

    def fork(self, seq: Sequence, n: int = 1) -> tuple[list[Sequence], list[tuple[int, int]]]:
        """n sequences that go on from a running one's tokens, on its blocks:
        (children, the block copies to make before the next step)."""
        if n < 1:
            raise ValueError(f"n must be >= 1, got {n}")
        if seq not in self.running:
            raise ValueError(f"sequence {seq.seq_id} is not running: only a running one has keys to share")
        if not self.block_manager.can_fork(seq, n):
            raise RuntimeError(f"no free blocks for {n} forks of sequence {seq.seq_id}")
        children, copies = [], []
        for _ in range(n):
            child = seq.fork()
            copies += self.block_manager.fork(seq, child)
            self.running.append(child)
            children.append(child)
        return children, copies

    def pack(self) -> list[tuple[int, int]]:
        """Move the blocks in use to the pool's start: the block copies to make
        before the next step."""
        copies = self.block_manager.pack()
        moved = dict(copies)
        for seq in self.running:
            seq.block_table = [moved.get(b, b) for b in seq.block_table]
        return copies

    def preempt(self, seq: Sequence) -> None:
        self.block_manager.deallocate(seq)
        seq.status = SequenceStatus.WAITING
        self.waiting.appendleft(seq)

    def postprocess(self, seqs: list[Sequence], token_ids: list[int]) -> None:
        """Append each sampled token; finish on EOS, max_tokens or
        max_model_length (engine/scheduler.py:79-95)."""
        for seq, token_id in zip(seqs, token_ids):
            seq.append_token(token_id)
            stop_eos = not seq.ignore_eos and token_id == self.eos
            stop_max_tokens = seq.num_completion_tokens >= seq.max_tokens
            stop_max_len = seq.max_model_length is not None and seq.num_tokens >= seq.max_model_length
            if stop_eos or stop_max_tokens or stop_max_len:
                seq.status = SequenceStatus.FINISHED
                self.block_manager.deallocate(seq)
                self.running.remove(seq)
