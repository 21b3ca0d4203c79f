"""The KV pool in 8 bits (HIP): writes, reads and decode attention over it.

Codes and scales are those of oracle.fp8.act_quant with a group of D, bit for
bit; rows read back are the fp32 product of code and scale rounded once to bf16,
bit for bit.  Decode tolerance, per output: a rounding to bf16 (half a step,
2^-8 of it) and 2^-12 of sum w |v| for fp32 scores, exponentials and sums
(|scale q.k| <= 16 here: an absolute error of some 2^-19 in a score, the same
relative one in its weight) and a weight held to 16 bits (2^-16)."""
import numpy as np
import pytest
import torch

from llm_from_scratch_amd import kernels as K
from oracle import fp8 as F
from oracle import paged_kv as P

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP8 = torch.float8_e4m3fn
HEADS = [(12, 4, 64), (8, 8, 64), (32, 8, 128), (8, 1, 128), (15, 3, 64), (14, 2, 128), (16, 16, 128), (10, 2, 64)]


def poisoned(NB, BS, Hkv, D):
    """Codes and scales that are all NaN."""
    c = torch.full((2, NB, BS, Hkv, D), 0x7F, dtype=torch.uint8, device=DEV).view(FP8)
    s = torch.full((2, NB, Hkv, BS), float("nan"), device=DEV)
    return c[0], c[1], s[0], s[1]


def filled(rng, lens, BS, Hkv, D, spare=3, wide=2, first_block=0, blocks=None):
    """A poisoned pool with random codes and scales in the rows of ``lens``
    tokens, tables, and each sequence's keys and values in 64 bits."""
    need = [-(-n // BS) for n in lens]
    NB = (sum(need) + spare + first_block) if blocks is None else blocks
    kc, vc, ks, vs = poisoned(NB, BS, Hkv, D)
    ids = first_block + rng.permutation(NB - first_block)
    bt = np.full((len(lens), max(need, default=0) + wide), -1, np.int32)
    seqs, at = [], 0
    for b, n in enumerate(lens):
        bt[b, :need[b]] = ids[at:at + need[b]]
        at += need[b]
        t = np.arange(n)
        blk, off = (torch.from_numpy(x).to(DEV) for x in (bt[b][t // BS].astype(np.int64), t % BS))
        both = []
        for cache, scale in ((kc, ks), (vc, vs)):
            x = torch.from_numpy(rng.standard_normal((n, Hkv, D)).astype(np.float32) * 120).to(DEV).clamp_(-448, 448)
            c, s = x.to(FP8), torch.from_numpy(rng.uniform(0.004, 0.02, (n, Hkv)).astype(np.float32)).to(DEV)
            cache.view(torch.uint8)[blk, off] = c.view(torch.uint8)
            scale[blk, :, off] = s
            both.append((c.double() * s.double()[..., None]).cpu().numpy())
        seqs.append(both)
    return (kc, vc, ks, vs), torch.from_numpy(bt).to(DEV), seqs


def queries(rng, B, Hq, D):
    q = torch.from_numpy(rng.standard_normal((B, Hq, D)).astype(np.float32)).to(torch.bfloat16).to(DEV)
    if B * Hq * D:
        q.view(-1)[::7] *= 2.0 ** -9  # far below the row's largest
    return q


def close(got, q, seqs, scale, what=""):
    got, q = got.double().cpu().numpy(), q.double().cpu().numpy()
    assert np.isfinite(got).all(), what
    for b, (k, v) in enumerate(seqs):
        o, a = P.window_attention(q[b:b + 1], k, v, [len(k) - 1], scale, len(k) + 1, 0)
        err, tol = np.abs(got[b] - o[0]), 2.0 ** -8 * np.abs(o[0]) + (2.0 ** -12 + 2.0 ** -16) * a[0] + 1e-30
        assert (err <= tol).all(), f"{what} row {b} of {len(k)}: worst {(err / tol).max():.3g}"


def lens_of(seqs):
    return torch.tensor([len(k) for k, _ in seqs], dtype=torch.int64, device=DEV)


def decode(q, pool, lens, bt, **kw):
    return K.paged_attention_decode(q, pool[0], pool[1], lens, bt, k_scale=pool[2], v_scale=pool[3], **kw)


# ----------------------------------------------------------- store and load --
def bits(t):
    return t.contiguous().view(torch.uint8).cpu().numpy()


@pytest.mark.parametrize("Hkv,D", [(4, 64), (8, 128), (3, 64), (1, 128), (16, 64)])
@pytest.mark.parametrize("T,BS", [(1, 16), (37, 48), (300, 256)])
@pytest.mark.parametrize("layout", ["plain", "fused", "odd"])
def test_store_is_act_quant_per_head(Hkv, D, T, BS, layout):
    rng = np.random.default_rng(T + Hkv + D)
    width = {"plain": Hkv * D, "fused": (4 + 2 * Hkv) * D, "odd": Hkv * D + 3}[layout]
    x = rng.standard_normal((2, T, width)).astype(np.float32) * np.exp(rng.uniform(-20, 20, (2, T, 1))).astype(np.float32)
    x[rng.random(x.shape) < 0.1] = 0
    x[:, T // 2, :D] = -0.0
    x[:, T - 1, :D] = 3e38
    both = torch.from_numpy(x).to(torch.bfloat16).to(DEV)
    at = 1 if layout == "odd" else width - Hkv * D
    key, value = (both[i, :, at:at + Hkv * D].unflatten(1, (Hkv, D)) for i in (0, 1))
    NB = -(-T // BS) + 2
    kc, vc, ks, vs = poisoned(NB, BS, Hkv, D)
    slots = rng.permutation(NB * BS)[:T].astype(np.int64)
    slots[rng.random(T) < 0.2] = -1
    slots[T // 3] = NB * BS + 5
    K.store_kvcache_fp8(key, value, kc, vc, ks, vs, torch.from_numpy(slots).to(DEV))
    for t, cache, scale in ((key, kc, ks), (value, vc, vs)):
        codes, s = F.act_quant(t.float().cpu().numpy().reshape(T, Hkv * D), block_size=D)
        want = np.full((NB * BS, Hkv, D), 0x7F, np.uint8)
        want_s = np.full((NB * BS, Hkv), np.nan, np.float32)
        ok = (slots >= 0) & (slots < NB * BS)
        want[slots[ok]], want_s[slots[ok]] = codes.reshape(T, Hkv, D)[ok], s.reshape(T, Hkv)[ok]
        assert np.array_equal(bits(cache).reshape(want.shape), want)
        got_s = scale.transpose(1, 2).reshape(NB * BS, Hkv).cpu().numpy()
        assert np.array_equal(got_s.view(np.uint32)[slots[ok]], want_s.view(np.uint32)[slots[ok]])
        assert np.array_equal(np.isnan(got_s), np.isnan(want_s))


@pytest.mark.parametrize("Hkv,D,T", [(4, 64, 10301), (8, 128, 2601), (3, 64, 16385), (33, 128, 700), (512, 64, 5)])
def test_store_many_tokens_and_heads(Hkv, D, T):
    """Several pieces a thread, and more heads than a workgroup has pieces for."""
    g = torch.Generator(device=DEV).manual_seed(T)
    key, value = (torch.randn(T, Hkv, D, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    NB, BS = -(-T // 16) + 1, 16
    pool = poisoned(NB, BS, Hkv, D)
    slots = torch.randperm(NB * BS, generator=g, device=DEV)[:T]
    K.store_kvcache_fp8(key, value, *pool, slots)
    for x, cache, scale in ((key, pool[0], pool[2]), (value, pool[1], pool[3])):
        codes, s = K.act_quant(x.view(T, Hkv * D), block_size=D)  # bit for bit the oracle's (tests/test_gpu_fp8.py)
        assert torch.equal(cache.view(torch.uint8).flatten(0, 1)[slots].view(T, -1), codes.view(torch.uint8))
        assert torch.equal(scale.transpose(1, 2).flatten(0, 1)[slots], s)
        assert int(torch.isnan(scale).sum()) == (NB * BS - T) * Hkv
    if Hkv == 512:
        with pytest.raises(ValueError, match="512 kv heads"):
            K.store_kvcache_fp8(key.repeat(1, 2, 1), value.repeat(1, 2, 1), *poisoned(1, 16, 1024, 64), slots)


@pytest.mark.parametrize("Hkv,D", [(4, 64), (8, 128), (3, 64), (1, 128)])
@pytest.mark.parametrize("BS", [16, 48, 256])
def test_load_is_the_rounded_product(Hkv, D, BS):
    rng = np.random.default_rng(BS + D + Hkv)
    lens = [0, 1, 300, BS, BS + 1, 0, 77, 0]
    pool, bt, seqs = filled(rng, lens, BS, Hkv, D)
    if BS < 300:
        bt[2, 1] = -1  # positions without a block
        for x in seqs[2]:
            x[BS:2 * BS] = 0
    bt[6, 0] = 10 ** 6
    for x in seqs[6]:
        x[:BS] = 0
    cu = torch.from_numpy(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)).to(DEV)
    total = sum(lens) + 5  # rows of no sequence
    strided = torch.full((bt.size(0), bt.size(1) + 3), -7, dtype=torch.int32, device=DEV)
    strided[:, :bt.size(1)] = bt
    for tables in (bt, strided[:, :bt.size(1)]):
        got = K.load_kvcache_fp8(*pool, tables, cu, total)
        for g, i in zip(got, (0, 1)):
            want = np.zeros((total, Hkv, D))
            want[:sum(lens)] = np.concatenate([s[i] for s in seqs])
            # a 4-bit code times a 24-bit scale: the fp32 product rounds once, then bf16 again
            want = torch.from_numpy(want.astype(np.float32)).to(torch.bfloat16)
            assert g.is_contiguous() and torch.equal(g.cpu().view(torch.int16), want.view(torch.int16))
    none = K.load_kvcache_fp8(*pool, bt[:0], cu[:1], 3)
    assert all((t == 0).all() and t.shape == (3, Hkv, D) for t in none)
    assert K.load_kvcache_fp8(*pool, bt, cu, 0)[0].shape == (0, Hkv, D)
    # more rows asked than there are blocks in the table: zeros
    long = torch.tensor([0, 40 * BS], dtype=torch.int32, device=DEV)
    got = K.load_kvcache_fp8(*pool, bt[4:5], long, 40 * BS)[0]
    assert (got[bt.size(1) * BS:] == 0).all()


def test_load_many_sequences():
    rng = np.random.default_rng(3)
    lens = rng.integers(0, 4, 3000).tolist()
    pool, bt, seqs = filled(rng, lens, 16, 1, 64)
    cu = torch.from_numpy(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)).to(DEV)
    got = K.load_kvcache_fp8(*pool, bt, cu, sum(lens))
    for g, i in zip(got, (0, 1)):
        want = torch.from_numpy(np.concatenate([s[i] for s in seqs]).astype(np.float32)).to(torch.bfloat16)
        assert torch.equal(g.cpu(), want)


# ------------------------------------------------------------------- decode --
@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("BS", [16, 32, 48, 64, 256])
def test_decode(Hq, Hkv, D, BS):
    rng = np.random.default_rng(Hq + D + BS)
    lens = [1, 0, 15, 16, 17, 64, 65, 129, 255, 256, 257, 600, 0, 1023]
    pool, bt, seqs = filled(rng, lens, BS, Hkv, D)
    q = queries(rng, len(lens), Hq, D)
    print(f"fp8 decode {Hq}/{Hkv}x{D} blocks of {BS}", flush=True)
    o = decode(q, pool, lens_of(seqs), bt)
    close(o, q, seqs, D ** -0.5)
    assert (o[1] == 0).all() and (o[12] == 0).all()
    # another scale, tables with a stride, one sequence alone
    strided = torch.full((bt.size(0), bt.size(1) + 5), 3, dtype=torch.int32, device=DEV)
    strided[:, :bt.size(1)] = bt
    close(decode(q, pool, lens_of(seqs), strided[:, :bt.size(1)], scale=0.3), q, seqs, 0.3, "strided")
    close(decode(q[13:], pool, lens_of(seqs)[13:], bt[13:]), q[13:], seqs[13:], D ** -0.5, "alone")


@pytest.mark.parametrize("Hq,Hkv,D", HEADS[:4])
def test_decode_one_token_gives_its_value(Hq, Hkv, D):
    rng = np.random.default_rng(1)
    pool, bt, seqs = filled(rng, [1, 1, 1], 16, Hkv, D)
    o = decode(queries(rng, 3, Hq, D), pool, lens_of(seqs), bt)
    want = np.repeat(np.stack([v[0] for _, v in seqs]), Hq // Hkv, axis=1)
    assert torch.equal(o.cpu(), torch.from_numpy(want.astype(np.float32)).to(torch.bfloat16))


@pytest.mark.parametrize("Hq,Hkv,D", [(16, 4, 64), (32, 8, 128)])
def test_decode_long_ragged(Hq, Hkv, D):
    rng = np.random.default_rng(D)
    lens = [20011, 1, 4096, 70, 9000, 0, 333, 12288]
    pool, bt, seqs = filled(rng, lens, 256, Hkv, D)
    q = queries(rng, len(lens), Hq, D)
    close(decode(q, pool, lens_of(seqs), bt), q, seqs, D ** -0.5)


@pytest.mark.parametrize("Hq,Hkv,D", HEADS[:3])
def test_decode_skips_blocks_outside_the_pool(Hq, Hkv, D):
    """Entries of -1, of -2^31 and past the pool add nothing; where no block is
    left the output is 0."""
    rng = np.random.default_rng(7)
    lens, BS = [200, 64, 500, 33], 32
    pool, bt, seqs = filled(rng, lens, BS, Hkv, D)
    q = queries(rng, 4, Hq, D)
    for b, cols in ((0, [0, 6]), (2, [1, 2, 3, 15]), (3, [0, 1])):
        for c, bad in zip(cols, (-1, -2 ** 31, 10 ** 6, 2 ** 31 - 1)):
            bt[b, c] = bad
        keep = np.array([t for t in range(lens[b]) if t // BS not in cols], int)
        seqs[b] = [x[keep] for x in seqs[b]]
    o = decode(q, pool, torch.tensor(lens, device=DEV), bt)
    close(o, q, seqs, D ** -0.5)
    assert (o[3] == 0).all()


def test_decode_sharp_and_flat_weights():
    """Scores far apart (one key holds nearly all weight) and all alike."""
    rng = np.random.default_rng(8)
    pool, bt, seqs = filled(rng, [700, 700], 64, 2, 64)
    q = queries(rng, 2, 6, 64)
    lens = lens_of(seqs)
    for scale in (0.0, 1e-6, 1.2):
        close(decode(q, pool, lens, bt, scale=scale), q, seqs, scale, f"scale {scale}")
    q[0] = 0
    close(decode(q, pool, lens, bt), q, seqs, 0.125, "no query")


@pytest.mark.parametrize("Hq,Hkv,D", [(12, 4, 64), (32, 8, 128), (14, 2, 64)])
def test_decode_quantised_output(Hq, Hkv, D):
    rng = np.random.default_rng(9)
    pool, bt, seqs = filled(rng, [300, 0, 2000, 17], 256, Hkv, D)
    q = queries(rng, 4, Hq, D)
    o, oq, os_ = decode(q, pool, lens_of(seqs), bt, quant=True)
    close(o, q, seqs, D ** -0.5)
    assert torch.equal(o, decode(q, pool, lens_of(seqs), bt))
    wq, ws = K.act_quant(o.view(4, -1))
    assert np.array_equal(bits(oq), bits(wq)) and torch.equal(os_, ws)


def test_decode_many_sequences():
    """More sequences than the balanced split holds."""
    rng = np.random.default_rng(10)
    B, Hq, Hkv, D = 9000, 4, 2, 64
    lens = rng.integers(0, 20, 64)
    pool, bt, seqs = filled(rng, lens.tolist(), 16, Hkv, D)
    q = queries(rng, B, Hq, D)
    at = torch.arange(B, device=DEV) % 64
    o = decode(q, pool, lens_of(seqs)[at], bt[at])
    rows = [0, 1, 63, 64, 4097, 8191, 8192, 8999]
    close(o[rows], q[rows], [seqs[r % 64] for r in rows], D ** -0.5)
    for lo in range(0, B, 3000):
        s = slice(lo, lo + 3000)
        diff = (o[s].float() - decode(q[s], pool, lens_of(seqs)[at][s], bt[at][s]).float()).abs().max()
        assert diff <= 0.05


@pytest.mark.parametrize("Hq,Hkv,D", [(10, 5, 64), (6, 6, 128), (14, 7, 64), (40, 10, 128), (9, 9, 64)])
@pytest.mark.parametrize("BS", [16, 64])
def test_decode_of_heads_that_fill_no_last_group(Hq, Hkv, D, BS):
    """Waves work on four kv heads at a time; in the last group some of them have
    none, for their whole share of the batch (one long sequence) or for a part of
    it (short ones)."""
    rng = np.random.default_rng(Hq + D + BS)
    for lens in ([5000], [1], [0, 1, 15, 65, 300, 0, 700, 64, 2049], rng.integers(1, 90, 70).tolist()):
        pool, bt, seqs = filled(rng, lens, BS, Hkv, D)
        q = queries(rng, len(lens), Hq, D)
        print(f"fp8 decode {Hq}/{Hkv}x{D} blocks of {BS}, {len(lens)} sequences", flush=True)
        o = decode(q, pool, lens_of(seqs), bt)
        close(o, q, seqs, D ** -0.5, f"{len(lens)} sequences")
        if Hq * D % 128 == 0:
            o2, oq, os_ = decode(q, pool, lens_of(seqs), bt, quant=True)
            wq, ws = K.act_quant(o.view(len(lens), -1))
            assert torch.equal(o, o2) and np.array_equal(bits(oq), bits(wq)) and torch.equal(os_, ws)


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 4, 128), (6, 3, 128), (5, 5, 64)])
def test_decode_many_sequences_of_several_heads(Hq, Hkv, D):
    """Past the balanced split's batches, with groups of three and four heads."""
    rng = np.random.default_rng(Hq + D)
    B = 8200
    lens = rng.integers(0, 70, 64)
    pool, bt, seqs = filled(rng, lens.tolist(), 16, Hkv, D)
    q = queries(rng, B, Hq, D)
    at = torch.arange(B, device=DEV) % 64
    o = decode(q, pool, lens_of(seqs)[at], bt[at])
    rows = list(range(64)) + [4097, 8191, 8192, 8199]
    close(o[rows], q[rows], [seqs[r % 64] for r in rows], D ** -0.5)


def test_decode_batches_of_none_and_short_tables():
    rng = np.random.default_rng(11)
    pool, bt, seqs = filled(rng, [40, 40], 16, 2, 64)
    q = queries(rng, 2, 4, 64)
    assert decode(q[:0], pool, lens_of(seqs)[:0], bt[:0]).shape == (0, 4, 64)
    # a context past its table is cut there
    cut = [[x[:32] for x in s] for s in seqs]
    close(decode(q, pool, lens_of(seqs) * 100, bt[:, :2]), q, cut, 0.125, "cut")
    assert (decode(q, pool, lens_of(seqs), bt[:, :0]) == 0).all()
    far = torch.tensor([2 ** 62, -2 ** 32 + 5], device=DEV)
    close(decode(q, pool, far, bt[:, :2]), q, [cut[0], [x[:0] for x in cut[1]]], 0.125, "far")
    close(decode(q, pool, -lens_of(seqs), bt), q, [[x[:0] for x in s] for s in seqs], 0.125, "below zero")


def test_pool_past_32_bits():
    """Codes and scales whose offsets pass 2^31 (and 2^32 bytes of bf16 rows)."""
    rng = np.random.default_rng(12)
    BS, Hkv, D, NB = 256, 8, 128, 8300
    assert (NB - 100) * BS * Hkv * D > 2 ** 31
    lens = [1000, 257]
    pool, bt, seqs = filled(rng, lens, BS, Hkv, D, first_block=NB - 50, blocks=NB)
    q = queries(rng, 2, 32, D)
    close(decode(q, pool, lens_of(seqs), bt), q, seqs, D ** -0.5)
    cu = torch.tensor([0, 1000, 1257], dtype=torch.int32, device=DEV)
    k, v = K.load_kvcache_fp8(*pool, bt, cu, 1257)
    want = torch.from_numpy(np.concatenate([s[0] for s in seqs]).astype(np.float32)).to(torch.bfloat16)
    assert torch.equal(k.cpu(), want)
    last = torch.tensor([NB * BS - 1], device=DEV)
    K.store_kvcache_fp8(k[:1], v[:1], *pool, last)
    codes, s = F.act_quant(k[:1].float().cpu().numpy().reshape(1, -1), block_size=D)
    assert np.array_equal(bits(pool[0][-1, -1]).reshape(-1), codes.reshape(-1))
    assert np.array_equal(pool[2][-1, :, -1].cpu().numpy(), s.reshape(-1))


def test_decode_in_graphs_and_on_streams():
    """Two captured decodes of different lengths, each with its own workspace,
    replayed in turn with eager work between; and a call on another stream."""
    rng = np.random.default_rng(13)
    Hq, Hkv, D = 12, 4, 64
    pool, bt, seqs = filled(rng, [3000, 500, 64, 1], 64, Hkv, D)
    q = queries(rng, 4, Hq, D)
    need = K.paged_decode_fp8_workspace_bytes(4, Hq, D)
    graphs = []
    for _ in range(2):
        ws = torch.empty(need, dtype=torch.uint8, device=DEV)
        lens = torch.zeros(4, dtype=torch.int64, device=DEV)
        decode(q, pool, lens, bt, workspace=ws)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o, oq, os_ = decode(q, pool, lens, bt, workspace=ws, quant=True)
        graphs.append((g, lens, o, oq, ws))  # a captured call's workspace lives as long as its graph
    full = lens_of(seqs)
    for turn in range(3):
        cuts = [torch.clamp(full - 17 * turn - 5 * i, min=0) for i in range(2)]
        for (g, lens, o, oq, _), n in zip(graphs, cuts):
            lens.copy_(n)
            g.replay()
        for (g, lens, o, oq, _), n in zip(graphs, cuts):
            assert torch.equal(o, decode(q, pool, n, bt))
            assert np.array_equal(bits(oq), bits(K.act_quant(o.view(4, -1))[0]))
    want = decode(q, pool, full, bt)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = decode(q, pool, full, bt)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_refusals():
    rng = np.random.default_rng(14)
    pool, bt, seqs = filled(rng, [40], 16, 2, 64)
    q, lens = queries(rng, 1, 4, 64), lens_of(seqs)
    kc, vc, ks, vs = pool
    with pytest.raises(ValueError, match="window"):
        decode(q, pool, lens, bt, window=4)
    with pytest.raises(AssertionError, match="go together"):
        K.paged_attention_decode(q, kc, vc, lens, bt, k_scale=ks)
    with pytest.raises(AssertionError, match="blocks_per_split"):
        decode(q, pool, lens, bt, blocks_per_split=1)
    with pytest.raises(TypeError, match="k_cache"):
        decode(q, (kc.to(torch.bfloat16), vc, ks, vs), lens, bt)
    with pytest.raises(AssertionError, match="k_scale"):
        decode(q, (kc, vc, ks.transpose(1, 2), vs), lens, bt)
    with pytest.raises(ValueError, match="workspace of"):
        decode(q, pool, lens, bt, workspace=torch.empty(16, dtype=torch.uint8, device=DEV))
    with pytest.raises(ValueError, match="runs? on the GPU|kernels run"):
        decode(q, pool, lens.cpu(), bt)
    with pytest.raises(TypeError, match="key"):
        K.store_kvcache_fp8(q[:, :2].float(), q[:, :2].float(), *pool, torch.zeros(1, dtype=torch.int64, device=DEV))
    with pytest.raises(AssertionError, match="slot_mapping"):
        K.store_kvcache_fp8(q[:, :2], q[:, :2], *pool, torch.zeros(2, dtype=torch.int64, device=DEV))
    with pytest.raises(TypeError, match="cu_seqlens"):
        K.load_kvcache_fp8(*pool, bt, torch.zeros(2, dtype=torch.int64, device=DEV), 4)
