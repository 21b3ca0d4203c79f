"""Sequence state, as engine/sequence.py of the reference (same attributes and
methods).  One behavioural fix: ``last_block_num_tokens`` is ``block_size``
(not 0) when the length is a positive multiple of the block size, so the
decode slot ``block_table[-1]*BS + last_block_num_tokens - 1`` and the
prefill slot list of a full last block are right (the reference returns 0,
engine/sequence.py:67-69, which points the decode slot into the previous
block and gives a full last block an empty slot list).
"""
from __future__ import annotations

import math
import operator
from array import array
from copy import copy
from dataclasses import dataclass
from enum import Enum, auto
from itertools import count
from typing import Optional

import numpy as np


PENALTY_LIMIT = 1e30  # finite logits stay finite in fp32 with penalties and biases up to it


def check_penalties(sp) -> tuple[Optional[dict[int, float]], Optional[np.ndarray]]:
    """logit_bias and allowed_token_ids as a Sequence holds them, checked with the
    penalties."""
    assert 0 < sp.repetition_penalty < math.inf, "repetition_penalty must be > 0"
    assert 1 / PENALTY_LIMIT <= sp.repetition_penalty <= PENALTY_LIMIT, \
        f"repetition_penalty must be in [{1 / PENALTY_LIMIT:g}, {PENALTY_LIMIT:g}]"
    assert abs(sp.presence_penalty) <= PENALTY_LIMIT and abs(sp.frequency_penalty) <= PENALTY_LIMIT, \
        f"presence_penalty and frequency_penalty must be finite, at most {PENALTY_LIMIT:g} in size"
    bias = allowed = None
    if sp.logit_bias:
        assert len(sp.logit_bias) <= 1024, "logit_bias holds at most 1024 tokens"
        bias = {operator.index(t): float(v) for t, v in sp.logit_bias.items()}
        assert all(-2 ** 31 <= t < 2 ** 31 for t in bias), "logit_bias tokens must fit 32 bits"
        assert all(abs(v) <= PENALTY_LIMIT or v == -math.inf for v in bias.values()), \
            f"logit_bias values must be at most {PENALTY_LIMIT:g} in size, or -infinity"
    if sp.allowed_token_ids is not None:
        ids = sp.allowed_token_ids
        if not (isinstance(ids, np.ndarray) and ids.dtype.kind in "iu"):
            ids = [operator.index(t) for t in ids]
            assert all(-2 ** 63 <= t < 2 ** 63 for t in ids), "allowed_token_ids must fit 64 bits"
        allowed = np.array(ids, np.int64)
        assert allowed.size > 0, "allowed_token_ids allows no token"
        assert allowed.ndim == 1, "allowed_token_ids must be one row"
    return bias, allowed


@dataclass
class SamplingParams:
    """utils/sampler.py:7-23 of the reference, plus the ``max_model_length``
    field engine/sequence.py:34 reads from it, the filters of
    kernels.sample_filtered (top_k 0, top_p 1 and min_p 0: none) and what
    kernels.apply_penalties does to the logits before: repetition_penalty
    (1: none) for tokens of the prompt and the completion, presence_penalty and
    frequency_penalty (0: none) for those of the completion, logit_bias (token ->
    value, -infinity for a token never drawn) and allowed_token_ids (None: all;
    a list, set or array of whole numbers).  Tokens outside the vocabulary are
    ignored, but one at least must be left to draw (Sequence.check_tokens)."""
    temperature: float = 1.0
    max_tokens: int = 256
    ignore_eos: bool = False
    max_model_length: Optional[int] = None
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    repetition_penalty: float = 1.0
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    logit_bias: Optional[dict[int, float]] = None
    allowed_token_ids: Optional[list[int]] = None

    def __post_init__(self):
        assert self.temperature > 1e-10, "greedy sampling is not permitted"
        assert 0 <= self.top_k < 2 ** 31 and 0 < self.top_p <= 1 and 0 <= self.min_p <= 1, \
            "top_k must be in [0, 2**31), top_p in (0, 1], min_p in [0, 1]"
        check_penalties(self)


class SequenceStatus(Enum):
    WAITING = auto()
    RUNNING = auto()
    FINISHED = auto()


class Sequence:
    block_size = 256
    counter = count()

    def __init__(self, token_ids: list[int], sampling_params: Optional[SamplingParams] = None):
        sp = sampling_params or SamplingParams()
        self.seq_id = next(Sequence.counter)
        self.status = SequenceStatus.WAITING
        self.token_ids = copy(token_ids)
        self.last_token = self.token_ids[-1] if self.token_ids else None
        self.num_tokens = len(self.token_ids)
        self.num_prompt_tokens = len(self.token_ids)
        self.num_cached_tokens = 0
        self.block_table: list[int] = []  # -1: a block freed behind the sliding window
        self.num_released_blocks = 0  # from the first block without sinks on
        self.top_k, self.top_p, self.min_p = sp.top_k, sp.top_p, sp.min_p
        self.repetition_penalty = sp.repetition_penalty
        self.presence_penalty, self.frequency_penalty = sp.presence_penalty, sp.frequency_penalty
        self.logit_bias, self.allowed_token_ids = check_penalties(sp)
        self._history = array("i")
        self.temperature = sp.temperature
        self.max_tokens = sp.max_tokens
        self.ignore_eos = sp.ignore_eos
        self.max_model_length = sp.max_model_length

    def fork(self) -> "Sequence":
        """A sequence of its own id that continues from the same tokens (its
        blocks still the parent's: BlockManager.fork)."""
        child = copy(self)
        child.seq_id = next(Sequence.counter)
        child.token_ids = copy(self.token_ids)
        child.block_table = copy(self.block_table)
        child._history = copy(self._history)
        return child

    def __len__(self):
        return self.num_tokens

    def __getitem__(self, idx):
        return self.token_ids[idx]

    @property
    def is_finished(self):
        return self.status == SequenceStatus.FINISHED

    @property
    def num_completion_tokens(self):
        return self.num_tokens - self.num_prompt_tokens

    @property
    def prompt_token_ids(self):
        return self.token_ids[:self.num_prompt_tokens]

    @property
    def completion_token_ids(self):
        return self.token_ids[self.num_prompt_tokens:]

    @property
    def num_cached_blocks(self):
        return int(math.ceil(self.num_cached_tokens / self.block_size))

    @property
    def num_blocks(self):
        return int(math.ceil(self.num_tokens / self.block_size))

    @property
    def last_block_num_tokens(self):
        """Tokens in the last (possibly full) block: num_tokens - (num_blocks-1)*BS."""
        if self.num_tokens == 0:
            return 0
        return self.num_tokens - (self.num_blocks - 1) * self.block_size

    def block(self, i):
        assert 0 <= i < self.num_blocks, f"Block index {i} out of range [0, {self.num_blocks})"
        return self.token_ids[i * self.block_size:(i + 1) * self.block_size]

    @property
    def has_penalties(self):
        return self.repetition_penalty != 1 or self.presence_penalty != 0 or self.frequency_penalty != 0

    def check_tokens(self, vocab: int) -> None:
        """Of ``vocab`` tokens, logit_bias and allowed_token_ids must leave one."""
        if not self.logit_bias and self.allowed_token_ids is None:
            return
        banned = {t for t, v in (self.logit_bias or {}).items() if v == -math.inf and 0 <= t < vocab}
        if self.allowed_token_ids is None:
            left = vocab > len(banned)
        else:
            ids = np.asarray(self.allowed_token_ids, np.int64)
            ids = ids[(ids >= 0) & (ids < vocab)]
            left = ids.size > 0 and (not banned or not banned.issuperset(ids.tolist()))
        if not left:
            raise ValueError(f"logit_bias and allowed_token_ids leave none of the {vocab} tokens")

    def history(self) -> np.ndarray:
        """The token ids as int32, from a copy that grows with them."""
        self._history.extend(self.token_ids[len(self._history):])
        return np.frombuffer(self._history, np.int32, self.num_tokens).copy()

    def append_token(self, token_id):
        self.token_ids.append(token_id)
        self.last_token = token_id
        self.num_tokens += 1
