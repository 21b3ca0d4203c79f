"""The operators together, as the engine runs them: a model with per-head norms
over a sliding window with sinks, its pool packed and branched while it runs,
filtered sampling.

Attention is checked teacher-forced, on the traced inputs of every layer: q and k
within one bf16 rounding (2^-8) of the float64 norm and rotation plus 2^-18 for
fp32, the attention output within the windowed attention's tolerance
(tests/test_gpu_window.py) of a float64 softmax over the pool's own rows.  What
must not change the arithmetic (where blocks lie, what freed ones hold,
branches beside a sequence, graph replay) is checked token for token."""
import numpy as np
import pytest
import torch

from llm_from_scratch_amd.context import reset_context
from llm_from_scratch_amd.decode_model import DecodeModel, DecodeModelConfig
from llm_from_scratch_amd.engine import BlockManager, LLMEngine, ModelRunner, Sampler, SamplingParams, Sequence
from llm_from_scratch_amd.engine.model_runner import prefill_parts
from oracle import paged_kv as P

pytestmark = pytest.mark.gpu
BS = 16
CFG = DecodeModelConfig(vocab_size=1024, d_model=256, num_layers=2, num_heads=4, num_kv_heads=2, d_ff=128,
                        n_routed_experts=4, num_experts_per_tok=2, max_model_length=512, sliding_window=50,
                        num_sink_tokens=3, qk_norm="head")


@pytest.fixture(autouse=True)
def block_size():
    old = Sequence.block_size
    Sequence.block_size = BS
    yield
    Sequence.block_size = old


def model_of(cfg, seed):
    model = DecodeModel(cfg, device="cuda", seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    for layer in model.layers:  # norm weights other than 1
        for norm in (layer.att.q_norm, layer.att.k_norm):
            norm.weight.data.copy_(1 + 0.3 * torch.randn(norm.weight.shape, generator=g, device="cuda"))
    return model


def check_layers(model, cfg, seqs, positions, blocks):
    """The trace of a forward over ``positions`` of each sequence (flattened in
    order); ``blocks``: each sequence's blocks of the positions it stored."""
    D, Hq, Hkv = cfg.head_dim, cfg.num_heads, cfg.num_kv_heads
    cs = model.rope.cos_sin_cached.double()
    for i, layer in enumerate(model.layers):
        tr, att = model.trace[i], layer.att
        qkv = tr["qkv"].double().view(-1, Hq + 2 * Hkv, D)
        at = 0
        for s, pos, table in zip(seqs, positions, blocks):
            n = len(pos)
            rows = qkv[at:at + n]
            p = torch.tensor(pos, device="cuda")
            c, sn = cs[p, None, :D // 2], cs[p, None, D // 2:]

            def turned(x, w):
                y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + att.q_norm.eps) * w.double()
                lo, hi = y[..., :D // 2], y[..., D // 2:]
                return torch.cat([lo * c - hi * sn, hi * c + lo * sn], -1), torch.cat([lo.abs() + hi.abs()] * 2, -1)

            q = tr["q"][0] if isinstance(tr["q"], tuple) else tr["q"]
            want, size = turned(rows[:, :Hq], att.q_norm.weight)
            assert ((q[at:at + n].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * size).all()
            last = pos[-1] + 1
            t = np.arange(last)
            seen = P.window_mask(pos, last, cfg.sliding_window, cfg.num_sink_tokens).any(0)
            ids = np.asarray(table)[t // BS]
            assert (ids[seen] >= 0).all()
            kv = [cache.double().cpu().numpy()[np.maximum(ids, 0), t % BS] for cache in (att.k_cache, att.v_cache)]
            want, size = turned(rows[:, Hq:Hq + Hkv], att.k_norm.weight)
            stored = torch.from_numpy(kv[0][pos]).cuda()
            assert ((stored - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * size).all()
            assert torch.equal(torch.from_numpy(kv[1][pos]).cuda(), rows[:, Hq + Hkv:])
            o, a = P.window_attention(q[at:at + n].double().cpu().numpy(), *kv, pos, D ** -0.5, cfg.sliding_window,
                                      cfg.num_sink_tokens)
            got = tr["att_o"].view(-1, Hq, D)[at:at + n].double().cpu().numpy()
            assert (np.abs(got - o) <= 2.0 ** -8 * np.abs(o) + (2.0 ** -8 + 2.0 ** -12) * a).all()
            at += n


@torch.inference_mode()
def test_layers_teacher_forced():
    """Whole prompts, a prompt behind a cached prefix, and decode steps over
    blocks freed behind the window."""
    model = model_of(CFG, 5)
    runner = ModelRunner(model, CFG.runner_config(block_size=BS, num_kv_blocks=96, enforce_eager=True))
    bm = BlockManager(96, BS, CFG.sliding_window, CFG.num_sink_tokens)
    rng = np.random.default_rng(1)
    seqs = [Sequence(rng.integers(0, 1024, n).tolist()) for n in (1, 49, 50, 130, 161)]

    def forward(batch, prefill):
        model.trace = {}
        ids, pos = runner.prepare_prefill(batch) if prefill else runner.prepare_decode(batch)
        logits = runner.run_model(ids, pos, prefill)
        reset_context()
        return logits

    for s in seqs:
        bm.allocate(s)
    forward(seqs, True)
    check_layers(model, CFG, seqs, [list(range(len(s))) for s in seqs], [s.block_table for s in seqs])
    later = Sequence(seqs[4].token_ids[:96] + rng.integers(0, 1024, 20).tolist())
    bm.allocate(later)
    assert later.num_cached_tokens == 96
    forward([later], True)
    check_layers(model, CFG, [later], [list(range(96, 116))], [later.block_table])
    seqs.append(later)
    for _ in range(20):
        for s in seqs:
            s.append_token(int(rng.integers(0, 1024)))
            bm.release_behind(s)
            bm.append(s)
        runner.kv_cache[:, :, list(bm.free_block_ids)] = float("nan")  # what nobody sees takes no part
        logits = forward(seqs, False)
        assert torch.isfinite(logits).all()
        check_layers(model, CFG, seqs, [[len(s) - 1] for s in seqs], [s.block_table for s in seqs])
    assert -1 in seqs[4].block_table


def engine(seed=7, cfg=CFG, **kw):
    config = cfg.runner_config(block_size=BS, num_kv_blocks=64, max_num_seqs=8, max_num_sequences=8,
                               max_num_batched_tokens=512, eos=-1)
    config.update(kw)
    return LLMEngine(model_of(cfg, seed), config, generator=torch.Generator(device="cuda").manual_seed(3))


PROMPTS = [np.random.default_rng(9).integers(0, 1024, n).tolist() for n in (5, 70, 33, 120)]
GREEDY = SamplingParams(top_k=1, max_tokens=60)


def test_packing_and_freed_blocks_change_no_token():
    want = engine().generate(PROMPTS, GREEDY)["token_ids"]
    assert [len(t) for t in want] == [60] * 4
    eng = engine()
    for p in PROMPTS:
        eng.add_prompt(p, GREEDY)
    done, moved = {}, 0
    while not eng.scheduler.is_finished():
        outputs, _, _ = eng.step()
        done.update(outputs)
        before = [list(s.block_table) for s in eng.scheduler.running]
        n = eng.pack_kv_cache()
        moved += [list(s.block_table) for s in eng.scheduler.running] != before
        eng.model_runner.kv_cache[:, :, n:] = float("nan")
    assert [done[k] for k in sorted(done)] == want and moved > 3
    assert len(eng.scheduler.block_manager.free_block_ids) == 64
    # eager steps pick the same tokens as the captured ones
    assert engine(enforce_eager=True).generate(PROMPTS, GREEDY)["token_ids"] == want


@pytest.mark.parametrize("at", [1, 4, 12, 13])
def test_branches_repeat_their_parent_when_greedy_and_leave_it_alone(at):
    """Forked after ``at`` steps: at a partly filled block and at a full one
    (33 tokens stored + 15 make 48)."""
    for prompt in (PROMPTS[2], PROMPTS[0][:4]):
        want = engine().generate([prompt], GREEDY)["token_ids"][0]
        eng = engine()
        eng.add_prompt(prompt, GREEDY)
        for _ in range(at):
            eng.step()
        parent = eng.scheduler.running[0].seq_id
        ids = eng.fork(parent, 3)
        ids += eng.fork(ids[0])
        done = {}
        while not eng.scheduler.is_finished():
            done.update(eng.step()[0])
        assert sorted(done) == sorted([parent] + ids)
        assert all(t == want for t in done.values())
        with pytest.raises(ValueError, match="no running sequence"):
            eng.fork(parent)


def test_branches_draw_their_own_tokens():
    eng = engine()
    eng.add_prompt(PROMPTS[1], SamplingParams(temperature=1.5, top_k=400, top_p=0.99, min_p=1e-4, max_tokens=30))
    eng.step()
    parent = eng.scheduler.running[0].seq_id
    eng.fork(parent, 5)
    done = {}
    while not eng.scheduler.is_finished():
        done.update(eng.step()[0])
    assert len(done) == 6 and len({tuple(t) for t in done.values()}) == 6
    assert len({t[0] for t in done.values()}) == 1  # sampled before the fork


def test_filters_mix_in_a_batch_and_seeds_repeat():
    """Sequences with and without filters in one batch; a top_k of 1 among them
    picks its most likely tokens; runs repeat."""
    def run():
        eng = engine()
        eng.add_prompt(PROMPTS[0], SamplingParams(temperature=0.9, max_tokens=25))
        eng.add_prompt(PROMPTS[3], SamplingParams(top_k=1, max_tokens=25))
        eng.add_prompt(PROMPTS[1], SamplingParams(top_p=0.8, min_p=0.01, max_tokens=25))
        done = {}
        while not eng.scheduler.is_finished():
            done.update(eng.step()[0])
        return [done[k] for k in sorted(done)]

    a = run()
    assert a == run() and [len(t) for t in a] == [25] * 3
    eng = engine()
    eng.add_prompt(PROMPTS[0], GREEDY)
    eng.add_prompt(PROMPTS[3], GREEDY)
    eng.add_prompt(PROMPTS[1], GREEDY)
    done = {}
    while not eng.scheduler.is_finished():
        done.update(eng.step()[0])
    assert done[sorted(done)[1]][:25] == a[1]


def test_filter_draws_advance_whatever_the_generator():
    """Calls with generators of two seeds in turn: no draw repeats, a second
    sampler draws the same."""
    logits = torch.zeros(8, 4096, dtype=torch.bfloat16, device="cuda")
    T, p = torch.ones(8, device="cuda"), torch.full((8,), 0.99, device="cuda")
    g = [torch.Generator(device="cuda").manual_seed(s) for s in (5, 6)]
    runs = []
    for _ in range(2):
        s = Sampler()
        runs.append([tuple(s(logits, T, g[i % 2], top_p=p).tolist()) for i in range(6)])
    assert runs[0] == runs[1] and len(set(runs[0])) == 6


def test_a_stream_outgrows_its_pool():
    """20 blocks hold 320 tokens; a sequence runs to 500 behind its window."""
    eng = engine(num_kv_blocks=20)
    out = eng.generate([PROMPTS[0]], SamplingParams(top_k=20, max_tokens=490))["token_ids"][0]
    assert len(out) == 490


@torch.inference_mode()
def test_parts_of_a_resumed_prefill_teacher_forced():
    """A sequence longer than the token budget, prefilled in parts: every layer
    of every part, over the keys that the parts before it left in the pool."""
    model = model_of(CFG, 6)
    runner = ModelRunner(model, CFG.runner_config(block_size=BS, num_kv_blocks=40, enforce_eager=True,
                                                  max_num_batched_tokens=72))
    rng = np.random.default_rng(2)
    s = Sequence(rng.integers(0, 1024, 9).tolist())
    for t in rng.integers(0, 1024, 250).tolist():
        s.append_token(t)
    BlockManager(40, BS, CFG.sliding_window, CFG.num_sink_tokens).allocate(s)
    parts = prefill_parts([s], BS, runner.token_budget())
    assert [p[0].num_tokens for p in parts] == [64, 128, 192, 256, 259]
    for part in parts:
        model.trace = {}
        runner.run_model(*runner.prepare_prefill(part), True)
        reset_context()
        pos = list(range(part[0].num_cached_tokens, part[0].num_tokens))
        check_layers(model, CFG, part, [pos], [s.block_table])


def test_streams_past_the_token_budget_are_resumed():
    """Streams of 200 tokens in a pool of 224, 64 tokens a prefill: all finish,
    and no prefill but of whole blocks within the budget."""
    eng = engine(num_kv_blocks=14, max_num_batched_tokens=64, enforce_eager=True)
    run_model, sizes, resumed = eng.model_runner.run_model, [], []

    def noted(ids, positions, is_prefill):
        if is_prefill:
            sizes.append(ids.numel())
            resumed.append(int(positions[0]) > 0)
        return run_model(ids, positions, is_prefill)

    eng.model_runner.run_model = noted
    out = eng.generate([p[:60] for p in PROMPTS], SamplingParams(top_k=20, max_tokens=200))["token_ids"]
    assert [len(t) for t in out] == [200] * 4
    assert max(sizes) <= 64 and any(resumed)
