"""paged_attention_decode_shared (HIP): decode for groups of sequences whose
first blocks are the same ones, against a float64 oracle per sequence.

Tolerance, per output: a rounding of the output to bf16 (half a step, 2^-8 of
it), a rounding of every weight to bf16 (2^-8 of sum w |v|, which bounds the
output too) and 2^-12 of that sum for fp32 scores, exponentials and sums
(|scale q.k| <= 16 here: an absolute error of some 2^-19 in a score, the same
relative one in its weight)."""
import numpy as np
import pytest
import torch

from llm_from_scratch_amd import kernels as K
from oracle import paged_kv as P

pytestmark = pytest.mark.gpu
DEV = "cuda"
HEADS = [(12, 4, 64), (8, 8, 64), (32, 8, 128), (8, 1, 128), (15, 3, 64), (14, 2, 128)]


def bf16(rng, *shape):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(torch.bfloat16).to(DEV)


def branches(rng, groups, BS, Hkv, D, spare=4, wide=2, first_block=0, blocks=None):
    """groups: [(shared blocks, [lengths])].  A pool that holds NaN in every row
    nobody sees, tables, lengths, (cu_groups, shared_blocks) and each sequence's
    keys and values in 64 bits."""
    lens = [n for _, g in groups for n in g]
    own = [max(0, -(-n // BS) - s) for s, g in groups for n in g]
    # a group's shared blocks: those that its longest sequence reaches into
    common = [min(s, -(-max(g, default=0) // BS)) for s, g in groups]
    NB = (sum(own) + sum(common) + spare + first_block) if blocks is None else blocks
    kc = torch.full((NB, BS, Hkv, D), float("nan"), device=DEV, dtype=torch.bfloat16)
    vc = kc.clone()
    ids = iter((first_block + rng.permutation(NB - first_block)).tolist())
    width = max([-(-n // BS) for n in lens] + [s for s, _ in groups], default=0) + wide
    bt = np.full((len(lens), width), -1, np.int32)
    seqs, b = [], 0
    for (s, g), c in zip(groups, common):
        head = [next(ids) for _ in range(c)]
        rows = min(s * BS, max(g, default=0))
        hk, hv = bf16(rng, rows, Hkv, D), bf16(rng, rows, Hkv, D)
        for i, blk in enumerate(head):
            n = min(BS, rows - i * BS)
            kc[blk, :n], vc[blk, :n] = hk[i * BS:i * BS + n], hv[i * BS:i * BS + n]
        for n in g:
            bt[b, :c] = head
            tail = max(0, n - s * BS)
            k, v = bf16(rng, tail, Hkv, D), bf16(rng, tail, Hkv, D)
            for i in range(-(-tail // BS)):
                blk = next(ids)
                bt[b, s + i] = blk
                m = min(BS, tail - i * BS)
                kc[blk, :m], vc[blk, :m] = k[i * BS:i * BS + m], v[i * BS:i * BS + m]
            seqs.append([torch.cat([h[:min(n, s * BS)], t]).double().cpu().numpy() for h, t in ((hk, k), (hv, v))])
            b += 1
    cu = np.concatenate([[0], np.cumsum([len(g) for _, g in groups])]).astype(np.int32)
    meta = [torch.from_numpy(x).to(DEV) for x in (cu, np.array([s for s, _ in groups], np.int32))]
    return kc, vc, torch.from_numpy(bt).to(DEV), torch.tensor(lens, dtype=torch.int64, device=DEV), meta, seqs


def close(got, q, seqs, scale, what=""):
    got, q = got.double().cpu().numpy(), q.double().cpu().numpy()
    assert np.isfinite(got).all(), what
    for b, (k, v) in enumerate(seqs):
        o, a = P.window_attention(q[b:b + 1], k, v, [len(k) - 1], scale, len(k) + 1, 0)
        err, tol = np.abs(got[b] - o[0]), 2.0 ** -8 * np.abs(o[0]) + (2.0 ** -8 + 2.0 ** -12) * a[0] + 1e-30
        assert (err <= tol).all(), f"{what} row {b} of {len(k)}: worst {(err / tol).max():.3g}"


def check(rng, groups, BS, Hq, Hkv, D, what="", **kw):
    kc, vc, bt, lens, meta, seqs = branches(rng, groups, BS, Hkv, D, **kw)
    q = bf16(rng, len(seqs), Hq, D)
    print(f"shared {Hq}/{Hkv}x{D} blocks of {BS} {what}", flush=True)
    o = K.paged_attention_decode_shared(q, kc, vc, lens, bt, *meta)
    close(o, q, seqs, D ** -0.5, what)
    return q, kc, vc, bt, lens, meta, seqs, o


@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("BS", [16, 48, 64, 256])
def test_groups(Hq, Hkv, D, BS):
    """Groups of one, none and many, prefixes of none and of many blocks,
    suffixes across tile edges, contexts that end among or before the shared
    blocks, and padding rows."""
    rng = np.random.default_rng(Hq + D + BS)
    for groups in (
        [(2, [2 * BS + n for n in (1, 15, 16, 17, 63, 64, 65, 130)])],
        [(0, [1, 100]), (3, [3 * BS + 7] * 3), (1, []), (5, [5 * BS + 300, 5 * BS, 5 * BS + 1]), (2, [2 * BS + 40])],
        [(3, [2 * BS + 5, 7, BS + 1]), (2, [BS + 15, BS + 3, 0])],
        [(4, [4 * BS + 9, 3 * BS, BS + 1, 1, 0, 4 * BS - 1, 5 * BS]), (1, [0, 0]), (2, [BS, 3])],
    ):
        check(rng, groups, BS, Hq, Hkv, D, str(groups)[:60])


@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
def test_large_groups(Hq, Hkv, D):
    """Groups whose rows fill several tiles, of sizes that leave ragged ones,
    behind a long prefix."""
    rng = np.random.default_rng(Hq * D)
    groups = [(33, (33 * 64 + rng.integers(0, 150, n)).tolist()) for n in (70, 1, 33)]
    check(rng, groups, 64, Hq, Hkv, D)


@pytest.mark.parametrize("Hq,Hkv,D", [(10, 5, 64), (6, 6, 128), (14, 7, 64), (40, 10, 128), (9, 9, 64)])
@pytest.mark.parametrize("BS", [16, 64])
def test_heads_that_fill_no_last_group(Hq, Hkv, D, BS):
    """Waves walk what sequences have for themselves four kv heads at a time; in
    the last group some of them have none, for their whole share (one long
    sequence) or for a part of it (short ones behind prefixes)."""
    rng = np.random.default_rng(Hq + D + BS)
    for groups in ([(0, [5000])], [(3, [3 * BS + 4000])], [(2, (2 * BS + rng.integers(1, 200, 9)).tolist()), (0, [1, 65])],
                   [(1, [BS + 70] * 40), (4, [4 * BS + 3] * 20)]):
        check(rng, groups, BS, Hq, Hkv, D, str(groups)[:60])


@pytest.mark.parametrize("Hq,Hkv,D", [(12, 4, 64), (32, 8, 128), (8, 1, 128)])
def test_weights_of_a_prefix_keep_16_bits(Hq, Hkv, D):
    """Values of either sign that nearly cancel show a weight's rounding beside
    the output's: no more than 2^-16 of sum w |v|, as over a pool in 8 bits, and
    2^-12 of it for fp32 scores, exponentials and sums."""
    rng = np.random.default_rng(Hq * D)
    for groups in ([(1, [16, 16, 5, 2])], [(4, [64, 64, 50, 80, 200])], [(130, [2080, 2080, 2090])]):
        kc, vc, bt, lens, meta, seqs = branches(rng, groups, 16, Hkv, D)
        vc.copy_(torch.where(vc > 0, 1.0, vc).where(~(vc < 0), -1.0))
        seqs = [[k, np.sign(v)] for k, v in seqs]
        q = bf16(rng, len(seqs), Hq, D)
        o = K.paged_attention_decode_shared(q, kc, vc, lens, bt, *meta).double().cpu().numpy()
        for b, (k, v) in enumerate(seqs):
            want, a = P.window_attention(q[b:b + 1].double().cpu().numpy(), k, v, [len(k) - 1], D ** -0.5, len(k) + 1, 0)
            err, tol = np.abs(o[b] - want[0]), 2.0 ** -8 * np.abs(want[0]) + (2.0 ** -12 + 2.0 ** -16) * a[0]
            assert (err <= tol).all(), f"{groups} row {b}: worst {(err / tol).max():.3g}"


def test_equals_the_plain_decode():
    """The same batch through paged_attention_decode, to the tolerance of both."""
    rng = np.random.default_rng(4)
    q, kc, vc, bt, lens, meta, seqs, o = check(rng, [(20, [5200, 5121, 6000]), (8, [2049] * 20)], 256, 32, 8, 128)
    plain = K.paged_attention_decode(q, kc, vc, lens, bt)
    assert ((o.float() - plain.float()).abs() <= 2.0 ** -6 * plain.float().abs() + 2.0 ** -8).all()
    # no groups, and rows of no group: nothing is shared
    none = torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(0, dtype=torch.int32, device=DEV)
    close(K.paged_attention_decode_shared(q, kc, vc, lens, bt, *none), q, seqs, 128 ** -0.5, "no groups")
    part = torch.tensor([3, 9], dtype=torch.int32, device=DEV), torch.tensor([8], dtype=torch.int32, device=DEV)
    close(K.paged_attention_decode_shared(q, kc, vc, lens, bt, *part), q, seqs, 128 ** -0.5, "one of the groups")


def test_blocks_outside_the_pool():
    """Entries of -1 and past the pool, among the shared blocks and after."""
    rng = np.random.default_rng(5)
    BS, groups = 32, [(6, [210, 400, 192, 100]), (4, [128, 129])]
    kc, vc, bt, lens, meta, seqs = branches(rng, groups, BS, 4, 64)
    q = bf16(rng, 6, 12, 64)
    bt[:4, 2], bt[:4, 5], bt[1, 8], bt[1, 12], bt[4:, :4] = -1, 10 ** 6, -5, 2 ** 31 - 1, -1
    gone = [[2, 5], [2, 5, 8, 12], [2, 5], [2, 5], [0, 1, 2, 3], [0, 1, 2, 3]]
    for b, cols in enumerate(gone):
        keep = np.array([t for t in range(int(lens[b])) if t // BS not in cols], int)
        seqs[b] = [x[keep] for x in seqs[b]]
    o = K.paged_attention_decode_shared(q, kc, vc, lens, bt, *meta)
    close(o, q, seqs, 0.125)
    assert (o[4] == 0).all()


def test_many_small_groups():
    rng = np.random.default_rng(6)
    groups = [(int(rng.integers(0, 4)), (rng.integers(0, 9, int(rng.integers(0, 4))) + 33).tolist()) for _ in range(300)]
    check(rng, groups, 16, 8, 2, 64)


def test_large_batches():
    """Thousands of sequences, in one group and in as many, up to the limit."""
    rng = np.random.default_rng(7)
    kc, vc, bt, lens, meta, seqs = branches(rng, [(3, (48 + rng.integers(0, 20, 64)).tolist())], 16, 2, 64)
    B = 8192
    at = torch.arange(B, device=DEV) % 64
    q = bf16(rng, B, 4, 64)
    rows = [0, 1, 63, 64, 4097, 8190, 8191]
    ones = torch.arange(B + 1, dtype=torch.int32, device=DEV), torch.full((B,), 3, dtype=torch.int32, device=DEV)
    one = torch.tensor([0, B], dtype=torch.int32, device=DEV), meta[1]
    for m in (one, ones):
        o = K.paged_attention_decode_shared(q, kc, vc, lens[at], bt[at], *m)
        close(o[rows], q[rows], [seqs[r % 64] for r in rows], 0.125)
        plain = K.paged_attention_decode(q, kc, vc, lens[at], bt[at])
        assert (o.float() - plain.float()).abs().max() <= 0.05


def test_groups_out_of_order_stay_in_bounds():
    """Boundaries past the batch, below zero and decreasing, shared blocks past
    the table and below zero: every access stays within the batch and its
    tables; where rows of no group are meant, nothing is shared."""
    rng = np.random.default_rng(8)
    kc, vc, bt, lens, meta, seqs = branches(rng, [(2, [100, 90, 80, 70])], 32, 2, 64)
    q = bf16(rng, 4, 4, 64)
    for cu, shared in (([0, 4, 9], [2, 3]), ([-3, 4], [2]), ([0, 4], [-1]), ([4, 0], [2])):
        m = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (cu, shared)]
        close(K.paged_attention_decode_shared(q, kc, vc, lens, bt, *m), q, seqs, 0.125, f"{cu} {shared}")
    m = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 2, 4], [99, 2])]
    o = K.paged_attention_decode_shared(q, kc, vc, lens, bt, *m)  # rows 0 and 1 are no branches of each other there
    close(o[2:], q[2:], seqs[2:], 0.125)
    close(o[:1], q[:1], seqs[:1], 0.125)


@pytest.mark.parametrize("Hq,Hkv,D", [(12, 4, 64), (32, 8, 128)])
def test_quantised_output(Hq, Hkv, D):
    rng = np.random.default_rng(9)
    q, kc, vc, bt, lens, meta, seqs, o = check(rng, [(3, [250, 192, 0, 400]), (0, [5])], 64, Hq, Hkv, D)
    o2, oq, os_ = K.paged_attention_decode_shared(q, kc, vc, lens, bt, *meta, quant=True)
    wq, ws = K.act_quant(o.view(5, -1))
    assert torch.equal(o, o2) and torch.equal(oq.view(torch.uint8), wq.view(torch.uint8)) and torch.equal(os_, ws)


def test_repeats_are_the_same_bits():
    rng = np.random.default_rng(10)
    q, kc, vc, bt, lens, meta, seqs, o = check(rng, [(40, (2560 + rng.integers(0, 900, 30)).tolist())], 64, 16, 4, 64)
    for _ in range(3):
        assert torch.equal(o, K.paged_attention_decode_shared(q, kc, vc, lens, bt, *meta))


def test_scale_stride_and_empty_batches():
    rng = np.random.default_rng(11)
    q, kc, vc, bt, lens, meta, seqs, o = check(rng, [(2, [100, 70, 64])], 32, 6, 2, 64)
    strided = torch.full((3, bt.size(1) + 5), 1, dtype=torch.int32, device=DEV)
    strided[:, :bt.size(1)] = bt
    close(K.paged_attention_decode_shared(q, kc, vc, lens, strided[:, :bt.size(1)], *meta, scale=0.3), q, seqs, 0.3)
    none = torch.zeros(2, dtype=torch.int32, device=DEV), meta[1]
    assert K.paged_attention_decode_shared(q[:0], kc, vc, lens[:0], bt[:0], *none).shape == (0, 6, 64)
    assert (K.paged_attention_decode_shared(q, kc, vc, lens, bt[:, :0], *meta) == 0).all()
    cut = [[x[:64] for x in s] for s in seqs]  # contexts past their tables are cut there
    close(K.paged_attention_decode_shared(q, kc, vc, lens * 50, bt[:, :2], *meta), q, cut, 0.125, "cut")
    assert (K.paged_attention_decode_shared(q, kc, vc, -lens, bt, *meta) == 0).all()
    far = torch.tensor([2 ** 62, -2 ** 32 + 5, 2 ** 33], device=DEV)
    close(K.paged_attention_decode_shared(q, kc, vc, far, bt[:, :2], *meta), q, [cut[0], [x[:0] for x in cut[1]], cut[2]], 0.125)


def test_pool_past_32_bits():
    rng = np.random.default_rng(12)
    NB, BS, Hkv, D = 4400, 256, 8, 128
    assert (NB - 100) * BS * Hkv * D > 2 ** 30
    check(rng, [(3, [800, 1000, 769]), (1, [300])], BS, 32, Hkv, D, first_block=NB - 40, blocks=NB)


def test_graphs_and_streams():
    """Two captured calls, each with its own workspace, whose groups and lengths
    change between replays, with eager work between; a call on another stream."""
    rng = np.random.default_rng(13)
    BS, Hq, Hkv, D = 64, 12, 4, 64
    kc, vc, bt, lens, meta, seqs = branches(rng, [(9, [700, 650, 577, 576]), (2, [300, 129, 128])], BS, Hkv, D)
    q = bf16(rng, 7, Hq, D)
    need = K.paged_decode_shared_workspace_bytes(7, 3, Hq, Hkv, D)
    plans = [([0, 4, 7, 7], [9, 2, 0]), ([0, 0, 4, 7], [1, 9, 1]), ([0, 2, 2, 4], [9, 0, 8]), ([0, 0, 0, 0], [0, 0, 0])]
    graphs = []
    for _ in range(2):
        ws = torch.empty(need, dtype=torch.uint8, device=DEV)
        state = [torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV),
                 torch.zeros_like(lens)]
        run = lambda: K.paged_attention_decode_shared(q, kc, vc, state[2], bt, *state[:2], workspace=ws)  # noqa: B023, E731
        run()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = run()
        graphs.append((g, state, o, ws))  # a captured call's workspace lives as long as its graph
    for turn in range(4):
        now = []
        for i, (g, state, o, _) in enumerate(graphs):
            plan = plans[(turn + i) % 4]
            now.append([torch.tensor(x, dtype=torch.int32, device=DEV) for x in plan] + [(lens - turn * 3 - i).clamp_(min=0)])
            for dst, src in zip(state, now[-1]):
                dst.copy_(src)
            g.replay()
        for (g, state, o, _), (cu, shared, n) in zip(graphs, now):
            assert torch.equal(o, K.paged_attention_decode_shared(q, kc, vc, n, bt, cu, shared))
            close(o, q, [[x[:int(m)] for x in s] for s, m in zip(seqs, n)], 0.125, f"turn {turn}")
    side = torch.cuda.Stream()
    want = K.paged_attention_decode_shared(q, kc, vc, lens, bt, *meta)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K.paged_attention_decode_shared(q, kc, vc, lens, bt, *meta)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_refusals():
    rng = np.random.default_rng(14)
    kc, vc, bt, lens, meta, seqs = branches(rng, [(1, [40, 50])], 16, 2, 64)
    q = bf16(rng, 2, 4, 64)
    call = K.paged_attention_decode_shared
    with pytest.raises(AssertionError, match="cu_groups"):
        call(q, kc, vc, lens, bt, meta[0][:1], meta[1])
    with pytest.raises(TypeError, match="shared_blocks"):
        call(q, kc, vc, lens, bt, meta[0], meta[1].long())
    with pytest.raises(TypeError, match="context_lens"):
        call(q, kc, vc, lens.int(), bt, *meta)
    with pytest.raises(ValueError, match="GPU"):
        call(q, kc, vc, lens, bt, meta[0].cpu(), meta[1])
    with pytest.raises(ValueError, match="workspace of"):
        call(q, kc, vc, lens, bt, *meta, workspace=torch.empty(16, dtype=torch.uint8, device=DEV))
    with pytest.raises(AssertionError, match="head_dim"):
        call(q[..., :32].contiguous(), kc, vc, lens, bt, *meta)
    with pytest.raises(ValueError, match="8192"):
        call(q.repeat(4097, 1, 1), kc, vc, lens.repeat(4097), bt.repeat(4097, 1), *meta)
