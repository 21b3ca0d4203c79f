"""Generation loop over the scheduler and the model runner, as
engine/llm_engine.py of the reference (step / add_prompt / generate).

One GPU, one process: the runner is called directly instead of through the
reference's worker processes and shared-memory RPC.  Prompts are token-id
lists; a tokenizer object (anything with ``encode``/``decode``) may be passed
for string prompts, since the reference's ``AutoTokenizer.from_pretrained``
fetches from the network.  ``step`` always returns three values (the
reference returns two when nothing is scheduled, :62-64).
"""
from __future__ import annotations

import time
from typing import Optional, Sequence as Seq, Union

import torch

from .. import kernels
from .model_runner import ModelRunner
from .scheduler import Scheduler
from .sequence import SamplingParams, Sequence


def check_window(model: torch.nn.Module, window: Optional[int], sinks: int) -> None:
    """The engine frees the blocks behind ``window`` but the first ``sinks``
    tokens': none of the model's attention layers may still see them.  Those
    are the modules that the runner gives their share of the pool; one without
    a ``window`` of its own sees everything."""
    if window is None:
        return
    kernels._window_args(window, sinks)
    for name, m in model.named_modules():
        if hasattr(m, "k_cache") and hasattr(m, "v_cache"):
            seen, first = getattr(m, "window", None), getattr(m, "sinks", 0)
            if seen is None or seen > window or first > sinks:
                raise ValueError(f"{name} sees a window of {seen} and {first} first tokens, but the engine keeps "
                                 f"{window} and {sinks}")


class LLMEngine:
    def __init__(self, model: torch.nn.Module, config: dict, tokenizer=None, device="cuda",
                 generator: Optional[torch.Generator] = None, verbose: bool = False):
        window, sinks = config.get("sliding_window"), config.get("num_sink_tokens", 0)
        check_window(model, window, sinks)
        self.model_runner = ModelRunner(model, config, device)
        block_size = config.get("block_size", 256)
        Sequence.block_size = block_size
        self.scheduler = Scheduler(
            max_num_sequences=config.get("max_num_sequences", config.get("max_num_seqs", 16)),
            max_num_batched_tokens=config.get("max_num_batched_tokens", 1024),
            max_cached_blocks=min(config.get("max_cached_blocks", self.model_runner.num_available_kv_blocks),
                                  self.model_runner.num_available_kv_blocks),
            block_size=block_size,
            eos=config.get("eos", 50256),
            sliding_window=window,
            num_sink_tokens=sinks)
        self.tokenizer = tokenizer
        self.generator = generator
        self.verbose = verbose

    def step(self):
        seqs, is_prefill = self.scheduler.schedule()
        if not seqs:
            return [], 0, is_prefill
        token_ids = self.model_runner.run(seqs, is_prefill, self.generator)
        self.scheduler.postprocess(seqs, token_ids)
        outputs = [(s.seq_id, s.completion_token_ids) for s in seqs if s.is_finished]
        n = sum(len(s) for s in seqs) if is_prefill else len(seqs)
        return outputs, n, is_prefill

    def add_prompt(self, prompt: Union[str, list[int]], sampling_params: SamplingParams) -> None:
        if isinstance(prompt, str):
            assert self.tokenizer is not None, "string prompts need a tokenizer"
            prompt = self.tokenizer.encode(prompt)
        self.scheduler.add_sequence(Sequence(list(prompt), sampling_params))

    def fork(self, seq_id: int, n: int = 1) -> list[int]:
        """n branches of a running sequence, between steps: each goes on from its
        tokens with draws of its own.  They share its blocks; only a partly
        filled last one is copied.  Returns their ids."""
        parent = next((s for s in self.scheduler.running if s.seq_id == seq_id), None)
        if parent is None:
            raise ValueError(f"no running sequence {seq_id}")
        children, copies = self.scheduler.fork(parent, n)
        self.model_runner.copy_blocks(copies)
        return [c.seq_id for c in children]

    def pack_kv_cache(self) -> int:
        """Move the blocks in use to the start of the pool, between steps;
        returns their number n: kv_cache[:, :, :n] then holds every running
        sequence's keys and values."""
        self.model_runner.copy_blocks(self.scheduler.pack())
        return len(self.scheduler.block_manager.used_block_ids)

    def generate(self, prompts: Seq[Union[str, list[int]]], sampling_params: SamplingParams) -> dict:
        for p in prompts:
            self.add_prompt(p, sampling_params)
        done: dict[int, list[int]] = {}
        while not self.scheduler.is_finished():
            t0 = time.perf_counter()
            outputs, n, is_prefill = self.step()
            if self.verbose:
                dt = time.perf_counter() - t0 + 1e-10
                print(f"{'prefill' if is_prefill else 'decode'}: {n} tokens, {n / dt:.1f} tokens/s")
            done.update(outputs)
        token_ids = [done[k] for k in sorted(done)]
        text = [self.tokenizer.decode(t) for t in token_ids] if self.tokenizer is not None else None
        return {"text": text, "token_ids": token_ids}
