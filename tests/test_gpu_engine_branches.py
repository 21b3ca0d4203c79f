"""The operators together, as the engine runs them: a pool in 8 bits, decode over
shared prefixes, penalties, biases and masks before the sampler.

Attention is checked teacher-forced, on the traced inputs of every layer, against
a float64 softmax over the pool's own rows, with the tolerance of each operator's
own tests; what the pool holds is checked bit for bit.  What must not change the
arithmetic (where blocks lie, branches beside a sequence, graph replay) is
checked token for token."""
import numpy as np
import pytest
import torch

from llm_from_scratch_amd import kernels as K
from llm_from_scratch_amd.context import reset_context
from llm_from_scratch_amd.decode_model import DecodeModel, DecodeModelConfig
from llm_from_scratch_amd.engine import BlockManager, LLMEngine, ModelRunner, SamplingParams, Sequence
from oracle import fp8 as F
from oracle import paged_kv as P

pytestmark = pytest.mark.gpu
BS = 16
FP8 = torch.float8_e4m3fn
CFG = DecodeModelConfig(vocab_size=1024, d_model=256, num_layers=2, num_heads=4, num_kv_heads=2, d_ff=128,
                        n_routed_experts=4, num_experts_per_tok=2, max_model_length=512)


@pytest.fixture(autouse=True)
def block_size():
    old = Sequence.block_size
    Sequence.block_size = BS
    yield
    Sequence.block_size = old


def engine(seed=7, **kw):
    config = CFG.runner_config(block_size=BS, num_kv_blocks=96, max_num_seqs=8, max_num_sequences=8,
                               max_num_batched_tokens=512, eos=-1)
    config.update(kw)
    return LLMEngine(DecodeModel(CFG, device="cuda", seed=seed), config,
                     generator=torch.Generator(device="cuda").manual_seed(3))


PROMPTS = [np.random.default_rng(9).integers(0, 1024, n).tolist() for n in (5, 70, 33, 120)]
GREEDY = SamplingParams(top_k=1, max_tokens=40)


def finish(eng):
    done = {}
    while not eng.scheduler.is_finished():
        done.update(eng.step()[0])
    return done


def rows_of(att, table, n):
    """Keys and values of n positions, in 64 bits, from the pool in either form."""
    t = np.arange(n)
    blk = torch.from_numpy(np.asarray(table, np.int64)[t // BS]).cuda()
    off = torch.from_numpy(t % BS).cuda()
    out = []
    for cache, scale in ((att.k_cache, att.k_scale), (att.v_cache, att.v_scale)):
        if scale is None:
            x = cache[blk, off].double()
        else:
            x = cache.view(torch.uint8)[blk, off].view(FP8).double() * scale[blk, :, off].double()[..., None]
        out.append(x.cpu().numpy())
    return out


def check_attention(model, seqs, queries, extra, rounded=False):
    """The traced attention of the last ``queries[i]`` tokens of each sequence
    over what the pool holds; extra: of sum w |v|, beside the output's rounding.
    rounded: over keys and values read back as bf16."""
    D, Hq = CFG.head_dim, CFG.num_heads
    for i, layer in enumerate(model.layers):
        tr, at = model.trace[i], 0
        q, o = tr["q"].view(-1, Hq, D).double().cpu().numpy(), tr["att_o"].view(-1, Hq, D).double().cpu().numpy()
        for s, m in zip(seqs, queries):
            n = s.num_tokens
            k, v = rows_of(layer.att, s.block_table, n)
            want, a = P.window_attention(q[at:at + m], k, v, np.arange(n - m, n), D ** -0.5, n + 1, 0)
            if rounded:  # v by 2^-8; k by as much, a score by that of scale sum |q k|, the weights by twice that
                heads = np.repeat(np.abs(k), Hq // k.shape[1], axis=1)
                score = np.einsum("mhd,nhd->mhn", np.abs(q[at:at + m]), heads).max() * D ** -0.5
                extra = 2.0 ** -8 * (2 + 2 * score) + 2.0 ** -12
            err = np.abs(o[at:at + m] - want)
            assert (err <= 2.0 ** -8 * np.abs(want) + extra * a + 1e-30).all(), (i, n, err.max())
            at += m


@torch.inference_mode()
def test_pool_in_8_bits_teacher_forced():
    """Whole prompts fill the pool with act_quant's codes and scales of the keys
    and values they computed; a prompt behind a cached prefix and decode steps
    attend over codes times scales."""
    model = DecodeModel(CFG, device="cuda", seed=5)
    runner = ModelRunner(model, CFG.runner_config(block_size=BS, num_kv_blocks=96, enforce_eager=True, kv_dtype=FP8))
    assert runner.kv_cache.dtype == FP8 and runner.kv_scales.shape == (2, 2, 96, 2, BS)
    runner.kv_scales.fill_(float("nan"))
    runner.kv_cache.view(torch.uint8).fill_(0x7F)
    bm = BlockManager(96, BS)
    rng = np.random.default_rng(1)
    seqs = [Sequence(rng.integers(0, 1024, n).tolist()) for n in (1, 49, 130, 161)]

    def forward(batch, prefill):
        model.trace = {}
        logits = runner.run_model(*(runner.prepare_prefill(batch) if prefill else runner.prepare_decode(batch)), prefill)
        reset_context()
        assert torch.isfinite(logits).all()

    for s in seqs:
        bm.allocate(s)
    forward(seqs, True)
    D, Hkv = CFG.head_dim, CFG.num_kv_heads
    for i, layer in enumerate(model.layers):
        qkv, at, att = model.trace[i]["qkv"], 0, layer.att
        pos = torch.cat([torch.arange(len(s), device="cuda") for s in seqs])
        _, k, v = K.qk_norm_rope_store(qkv, att.q_norm.weight, att.k_norm.weight, att.rope.cos_sin_cached, pos,
                                       CFG.num_heads, Hkv, att.q_norm.eps, return_kv=True)
        for s in seqs:
            n = len(s)
            for x, got in zip((k, v), rows_of(att, s.block_table, n)):
                codes, sc = F.act_quant(x[at:at + n].float().cpu().numpy().reshape(n, -1), block_size=D)
                want = torch.from_numpy(codes).view(FP8).double().numpy().reshape(n, Hkv, D) * sc.astype(np.float64)[..., None]
                assert np.array_equal(got, want)
            at += n
    later = Sequence(seqs[3].token_ids[:96] + rng.integers(0, 1024, 20).tolist())
    bm.allocate(later)
    assert later.num_cached_tokens == 96
    forward([later], True)
    check_attention(model, [later], [20], 0, rounded=True)
    seqs.append(later)
    for _ in range(20):
        for s in seqs:
            s.append_token(int(rng.integers(0, 1024)))
            bm.append(s)
        forward(seqs, False)
        check_attention(model, seqs, [1] * len(seqs), 2.0 ** -12 + 2.0 ** -16)


def test_pool_in_8_bits_moves_and_branches():
    """Packed after every step, in graphs and eagerly, and with branches beside
    it, a greedy sequence is the same."""
    eng = engine(kv_dtype=FP8)
    want = eng.generate(PROMPTS, GREEDY)["token_ids"]
    assert [len(t) for t in want] == [40] * 4
    assert engine(kv_dtype=FP8, enforce_eager=True).generate(PROMPTS, GREEDY)["token_ids"] == want
    eng = engine(kv_dtype=FP8)
    for p in PROMPTS:
        eng.add_prompt(p, GREEDY)
    done, moved = {}, 0
    while not eng.scheduler.is_finished():
        done.update(eng.step()[0])
        before = [list(s.block_table) for s in eng.scheduler.running]
        n = eng.pack_kv_cache()
        moved += [list(s.block_table) for s in eng.scheduler.running] != before
        eng.model_runner.kv_scales[:, :, n:] = float("nan")
        eng.model_runner.kv_cache.view(torch.uint8)[:, :, n:] = 0x7F
    assert [done[k] for k in sorted(done)] == want
    for at in (1, 7, 12):
        eng = engine(kv_dtype=FP8)
        eng.add_prompt(PROMPTS[1], GREEDY)
        for _ in range(at):
            eng.step()
        eng.fork(eng.scheduler.running[0].seq_id, 3)
        done = finish(eng)
        assert len(done) == 4 and len({tuple(t) for t in done.values()}) == 1


def test_pool_in_8_bits_is_sized_and_resumed():
    cfg = CFG.runner_config(block_size=BS, max_num_seqs=4, max_num_batched_tokens=512, enforce_eager=True,
                            gpu_memory_utilization=0.01)
    half, full = (ModelRunner(DecodeModel(CFG, device="cuda", seed=5), dict(cfg, kv_dtype=t)) for t in (FP8, torch.bfloat16))
    per = [r.kv_cache[:, :, 0].numel() * r.kv_cache.element_size() + (0 if r.kv_scales is None else
           r.kv_scales[:, :, 0].numel() * 4) for r in (half, full)]
    assert per == [2 * 2 * BS * 2 * 68, 2 * 2 * BS * 2 * 128] and half.num_available_kv_blocks > 1000
    # preempted sequences come back through their cached prefixes
    out = engine(kv_dtype=FP8, num_kv_blocks=14, max_num_batched_tokens=64,
                 enforce_eager=True).generate([p[:60] for p in PROMPTS], SamplingParams(top_k=20, max_tokens=150))
    assert [len(t) for t in out["token_ids"]] == [150] * 4


@torch.inference_mode()
def test_shared_prefixes_teacher_forced():
    """Branches of two sequences and a third alone, over 20 steps."""
    model = DecodeModel(CFG, device="cuda", seed=6)
    runner = ModelRunner(model, CFG.runner_config(block_size=BS, num_kv_blocks=96, enforce_eager=True,
                                                  share_prefixes=True))
    bm = BlockManager(96, BS)
    rng = np.random.default_rng(2)
    seqs = []
    for n, forks in ((70, 3), (33, 0), (130, 2)):
        s = Sequence(rng.integers(0, 1024, n).tolist())
        bm.allocate(s)
        runner.run_model(*runner.prepare_prefill([s]), True)
        s.append_token(int(rng.integers(0, 1024)))
        bm.append(s)
        seqs.append(s)
        for _ in range(forks):
            child = s.fork()
            runner.copy_blocks(bm.fork(s, child))
            seqs.append(child)
    for step in range(20):
        model.trace = {}
        ids = runner.prepare_decode(seqs)
        from llm_from_scratch_amd.context import get_context
        ctx = get_context()
        assert ctx.cu_groups.tolist() == [0, 4, 5, 8] and ctx.shared_blocks.tolist() == [4, 0, 8]
        logits = runner.run_model(*ids, False)
        reset_context()
        assert torch.isfinite(logits).all()
        check_attention(model, seqs, [1] * 8, 2.0 ** -8 + 2.0 ** -12)
        for s in seqs:
            s.append_token(int(rng.integers(0, 1024)))
            bm.append(s)


def test_shared_prefixes_in_graphs():
    """Groups that come, grow and go between replays: graphs and eager steps
    draw the same tokens, and greedy branches repeat their parent."""
    runs = []
    for eager in (False, True):
        eng = engine(share_prefixes=True, enforce_eager=eager)
        for p in PROMPTS[1:]:
            eng.add_prompt(p, SamplingParams(top_k=1, max_tokens=30))
        eng.step()
        ids = [s.seq_id for s in eng.scheduler.running]
        first = eng.fork(ids[2], 2)
        for _ in range(5):
            eng.step()
        more = eng.fork(first[0], 2)
        done = finish(eng)
        assert len({tuple(done[i]) for i in [ids[2], *first, *more]}) == 1
        runs.append([done[i] for i in sorted(done)])
    assert runs[0] == runs[1] and [len(t) for t in runs[0]] == [30] * 7


def test_penalties_biases_and_masks_in_the_engine():
    """A mask lets only its tokens through, a large frequency penalty repeats no
    token before all are used, a bias forces one, and a sequence without any is
    as if alone."""
    allowed = list(range(100, 150))
    eng = engine(num_kv_blocks=64)
    eng.add_prompt(PROMPTS[0], SamplingParams(top_k=1, max_tokens=40, allowed_token_ids=allowed, frequency_penalty=1e4))
    eng.add_prompt(PROMPTS[2], GREEDY)
    eng.add_prompt(PROMPTS[1], SamplingParams(temperature=5.0, max_tokens=40, logit_bias={77: 1e5}))
    eng.add_prompt(PROMPTS[3], SamplingParams(top_k=1, max_tokens=40, repetition_penalty=1e6, presence_penalty=1e4))
    done = finish(eng)
    masked, plain, biased, fresh = (done[k] for k in sorted(done))
    assert sorted(masked) == sorted(set(masked)) and set(masked) <= set(allowed)
    assert biased == [77] * 40
    assert len(set(fresh)) == 40
    assert plain == engine(num_kv_blocks=64).generate([PROMPTS[0], PROMPTS[2]], GREEDY)["token_ids"][1]


def test_all_together():
    """A pool in 8 bits with penalties, masks and forks, sampled: runs repeat."""
    runs = []
    for _ in range(2):
        eng = engine(kv_dtype=FP8)
        eng.add_prompt(PROMPTS[3], SamplingParams(temperature=1.2, top_p=0.9, repetition_penalty=1.3, frequency_penalty=0.4,
                                                  max_tokens=30, allowed_token_ids=list(range(0, 1024, 2))))
        eng.add_prompt(PROMPTS[3][:64] + PROMPTS[0], SamplingParams(temperature=0.8, min_p=0.01, max_tokens=30))
        eng.step()
        eng.fork(eng.scheduler.running[0].seq_id, 3)
        done = finish(eng)
        runs.append([done[k] for k in sorted(done)])
    assert runs[0] == runs[1] and len(runs[0]) == 5
    for t in [runs[0][0]] + runs[0][2:]:
        assert all(x % 2 == 0 for x in t)
