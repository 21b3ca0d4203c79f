"""Attention over a sliding window with sinks (HIP): prefill and decode, against
a float64 oracle on the same bf16 inputs.

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


def f64(t):
    return t.double().cpu().numpy()


def close(got, want, what):
    o, a = want
    err, tol = np.abs(f64(got) - o), 2.0 ** -8 * np.abs(o) + (2.0 ** -8 + 2.0 ** -12) * a + 1e-30
    assert np.isfinite(f64(got)).all(), what
    assert (err <= tol).all(), f"{what}: {np.argwhere(err > tol)[:3].tolist()} worst {(err / tol).max():.3g}"


def bf16(rng, *shape):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(torch.bfloat16).to(DEV)


def paged(rng, lens, firsts, BS, Hkv, D, sinks, spare=5, wide=2):
    """A pool whose unused blocks, hidden rows and rows past the contexts hold
    NaN, tables with -1 for every block that holds no visible key, and the
    sequences' keys and values [(K, V)]."""
    need = [-(-n // BS) for n in lens]
    NB = sum(need) + spare
    ids = rng.permutation(NB)
    kc = torch.full((NB, BS, Hkv, D), float("nan"), device=DEV, dtype=torch.bfloat16)
    vc = kc.clone()
    bt = np.full((len(lens), max(need, default=0) + wide), -1, np.int32)
    seqs, at = [], 0
    for b, (n, first) in enumerate(zip(lens, firsts)):
        k, v = bf16(rng, n, Hkv, D), bf16(rng, n, Hkv, D)
        seen = (np.arange(n) < sinks) | (np.arange(n) >= first)
        for i in range(need[b]):
            rows = np.arange(i * BS, min(n, (i + 1) * BS))
            rows = rows[seen[rows]]
            if len(rows):
                bt[b, i] = ids[at]
                kc[ids[at], rows - i * BS] = k[rows]
                vc[ids[at], rows - i * BS] = v[rows]
            at += 1
        seqs.append((f64(k), f64(v)))
    return kc, vc, torch.from_numpy(bt).to(DEV), seqs


HEADS = [(12, 4, 64), (8, 8, 64), (32, 8, 128), (8, 1, 128), (15, 3, 64), (14, 2, 128)]
WINDOWS = [(1, 0), (1, 3), (17, 0), (64, 4), (100, 70), (130, 1), (5000, 9)]


@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_prefill_whole_prompts(Hq, Hkv, D, window, sinks):
    rng = np.random.default_rng(Hq + D + window)
    lens = [1, 0, 15, 64, 65, 129, 300, 513]
    cu = np.concatenate([[0], np.cumsum(lens)])
    q, k, v = bf16(rng, cu[-1], Hq, D), bf16(rng, cu[-1], Hkv, D), bf16(rng, cu[-1], Hkv, D)
    cud = torch.from_numpy(cu.astype(np.int32)).to(DEV)
    o = K.flash_attn_varlen_func(q, k, v, cud, cud, max(lens), max(lens), window=window, sinks=sinks)
    for i, n in enumerate(lens):
        s = slice(cu[i], cu[i + 1])
        close(o[s], P.window_attention(f64(q[s]), f64(k[s]), f64(v[s]), np.arange(n), D ** -0.5, window, sinks),
              f"prompt of {n}")


@pytest.mark.parametrize("Hq,Hkv,D", HEADS[:4])
@pytest.mark.parametrize("BS", [16, 48, 256])
@pytest.mark.parametrize("window,sinks", [(1, 0), (33, 5), (21, 5), (200, 0), (257, 64), (100, 300), (645, 250)])
def test_prefill_chunks_over_the_pool(Hq, Hkv, D, BS, window, sinks):
    """New tokens behind cached ones; blocks behind the first query's window
    are freed and everything nobody sees is NaN."""
    rng = np.random.default_rng(BS + window + D)
    lens, new = [700, 64, 1, 901, 260, 33], [130, 64, 1, 1, 259, 7]
    kc, vc, bt, seqs = paged(rng, lens, [n - m - window + 1 for n, m in zip(lens, new)], BS, Hkv, D, sinks)
    cq, ck = (torch.from_numpy(np.concatenate([[0], np.cumsum(x)]).astype(np.int32)).to(DEV) for x in (new, lens))
    q = bf16(rng, sum(new), Hq, D)
    o = K.flash_attn_varlen_func(q, kc, vc, cq, ck, max(new), max(lens), 0.11, block_table=bt, window=window, sinks=sinks)
    at = 0
    for n, m, (k, v) in zip(lens, new, seqs):
        close(o[at:at + m], P.window_attention(f64(q[at:at + m]), k, v, np.arange(n - m, n), 0.11, window, sinks),
              f"{m} new of {n}")
        at += m


def test_prefill_queries_before_the_first_key_see_nothing():
    """lq > lk puts the first queries at positions below 0."""
    rng = np.random.default_rng(3)
    q, k, v = bf16(rng, 40, 4, 64), bf16(rng, 25, 2, 64), bf16(rng, 25, 2, 64)
    cq, ck = torch.tensor([0, 40], dtype=torch.int32, device=DEV), torch.tensor([0, 25], dtype=torch.int32, device=DEV)
    o = K.flash_attn_varlen_func(q, k, v, cq, ck, 40, 25, window=7, sinks=2)
    close(o, P.window_attention(f64(q), f64(k), f64(v), np.arange(-15, 25), 0.125, 7, 2), "short context")
    assert (o[:15] == 0).all()
    none = torch.zeros(2, dtype=torch.int32, device=DEV)
    o = K.flash_attn_varlen_func(q, k[:0], v[:0], cq, none, 40, 0, window=7, sinks=2)
    assert o.shape == q.shape and (o == 0).all()


@pytest.mark.parametrize("D", [64, 128])
def test_prefill_window_past_the_context_is_the_causal_attention(D):
    rng = np.random.default_rng(D)
    lens = [700, 3, 128]
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=DEV)
    q, k, v = bf16(rng, sum(lens), 8, D), bf16(rng, sum(lens), 2, D), bf16(rng, sum(lens), 2, D)
    a = K.flash_attn_varlen_func(q, k, v, cu, cu, max(lens), max(lens))
    for window, sinks in [(700, 0), (2 ** 40, 2 ** 40), (1, 700)]:
        b = K.flash_attn_varlen_func(q, k, v, cu, cu, max(lens), max(lens), window=window, sinks=sinks)
        scale = a.float().abs().mean().item()
        assert (a.float() - b.float()).abs().max().item() < 2.0 ** -7 * (scale + a.float().abs().max().item())


def test_prefill_large_scores_and_more_rows_than_max():
    """Scores to +-10^4 (one key takes all), and infinite q: NaN as a softmax over it."""
    rng = np.random.default_rng(11)
    q, k, v = bf16(rng, 200, 4, 64) * 40, bf16(rng, 200, 4, 64) * 40, bf16(rng, 200, 4, 64)
    cu = torch.tensor([0, 200], dtype=torch.int32, device=DEV)
    o = K.flash_attn_varlen_func(q, k, v, cu, cu, 200, 200, window=50, sinks=3)
    want, _ = P.window_attention(f64(q), f64(k), f64(v), np.arange(200), 0.125, 50, 3)
    # scores are near 10^3: fp32 leaves 2^-12 of them, so only rows whose first two differ by more are compared
    mask = P.window_mask(np.arange(200), 200, 50, 3)
    s = np.einsum("qhd,khd->hqk", f64(q), f64(k)) * 0.125
    s = np.sort(np.where(mask[None], s, -np.inf), -1)
    clear = ((s[..., -1] - s[..., -2]) > 20).T
    assert clear.mean() > 0.5 and np.abs(f64(o) - want)[clear].max() < 2.0 ** -7 * np.abs(want).max()
    q[100, 1] = float("inf")
    o = K.flash_attn_varlen_func(q, k, v, cu, cu, 200, 200, window=50, sinks=3)
    assert torch.isnan(o[100, 1]).all() and torch.isfinite(o[101]).all() and torch.isfinite(o[100, 0]).all()


@pytest.mark.parametrize("Hq,Hkv,D", HEADS)
@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("BS", [16, 48, 256])
def test_decode(Hq, Hkv, D, window, sinks, BS):
    rng = np.random.default_rng(BS + window + D + Hq)
    lens = [0, 1, 2, 16, 63, 64, 65, 131, 500, 1023, 17]
    kc, vc, bt, seqs = paged(rng, lens, [n - window for n in lens], BS, Hkv, D, sinks)
    q = bf16(rng, len(lens), Hq, D)
    cl = torch.tensor(lens, device=DEV)
    o = K.paged_attention_decode(q, kc, vc, cl, bt, window=window, sinks=sinks)
    for b, (n, (k, v)) in enumerate(zip(lens, seqs)):
        if n == 0:
            assert (o[b] == 0).all()
        else:
            close(o[b:b + 1], P.window_attention(f64(q[b:b + 1]), k, v, [n - 1], D ** -0.5, window, sinks), f"context {n}")


@pytest.mark.parametrize("B,Hq,Hkv,D,window,sinks", [(1, 12, 4, 64, 1024, 4), (3, 32, 8, 128, 4096, 16),
                                                   (70, 16, 4, 64, 1000, 4), (140, 8, 4, 64, 200, 0),
                                                   (300, 4, 1, 128, 333, 70), (64, 8, 8, 128, 64, 1)])
def test_decode_batches(B, Hq, Hkv, D, window, sinks):
    """Every way of splitting the work: few and many sequences, long windows,
    contexts from none to far past the window; the quantised output too."""
    rng = np.random.default_rng(B)
    lens = [int(x) for x in rng.integers(0, 3 * window, B)]
    lens[-1] = 2 * window + 3
    BS = 64
    kc, vc, bt, seqs = paged(rng, lens, [n - window for n in lens], BS, Hkv, D, sinks)
    q = bf16(rng, B, Hq, D)
    cl = torch.tensor(lens, device=DEV)
    o, oq, os_ = K.paged_attention_decode(q, kc, vc, cl, bt, 0.1, quant=True, window=window, sinks=sinks)
    same = K.paged_attention_decode(q, kc, vc, cl, bt, 0.1, window=window, sinks=sinks)
    for b, (n, (k, v)) in enumerate(zip(lens, seqs)):
        want = P.window_attention(f64(q[b:b + 1]), k, v, [n - 1], 0.1, window, sinks) if n else (np.zeros(1), np.zeros(1))
        close(o[b:b + 1], want, f"context {n}")
        close(same[b:b + 1], want, f"context {n}, no quantised output")
    wq, ws = K.act_quant(o.view(B, -1))
    assert torch.equal(oq.view(torch.uint8), wq.view(torch.uint8)) and torch.equal(os_, ws)


@pytest.mark.parametrize("B,Hq,Hkv,D,BS,window,sinks", [(45, 12, 4, 64, 16, 810, 4), (47, 32, 8, 128, 16, 790, 33),
                                                       (70, 8, 8, 64, 16, 520, 0), (33, 8, 4, 64, 64, 4100, 70),
                                                       (300, 8, 1, 128, 32, 1601, 1)])
def test_decode_long_windows_of_many_sequences(B, Hq, Hkv, D, BS, window, sinks):
    """An equal share of all visible tiles per workgroup: contexts of none, one,
    a window's length and far past it; also captured, with other lengths and
    tables at each replay, and with the quantised output."""
    rng = np.random.default_rng(B)
    NB, width = 300, 2 * window // BS + 3
    kc, vc, q = bf16(rng, NB, BS, Hkv, D), bf16(rng, NB, BS, Hkv, D), bf16(rng, B, Hq, D)
    fk, fv = f64(kc), f64(vc)

    def contexts():
        lens = rng.integers(0, width * BS + 1, B)
        lens[:6] = 0, 1, window, window + 1, window + sinks, width * BS
        return torch.from_numpy(lens).to(DEV), torch.from_numpy(rng.integers(0, NB, (B, width)).astype(np.int32)).to(DEV)

    cl, bt = contexts()
    call = lambda: K.paged_attention_decode(q, kc, vc, cl, bt, 0.1, quant=True, window=window, sinks=sinks)
    o, oq, os_ = call()
    wq, ws = K.act_quant(o.view(B, -1))
    assert torch.equal(oq.view(torch.uint8), wq.view(torch.uint8)) and torch.equal(os_, ws)
    for b in list(range(8)) + list(range(8, B, 1 + B // 8)) + [B - 1]:
        n, table = int(cl[b]), bt[b].cpu().numpy()
        keep = np.flatnonzero(P.window_mask([n - 1], n, window, sinks)[0]) if n else np.zeros(0, int)
        slots = table[keep // BS], keep % BS
        want = P.window_attention(f64(q[b:b + 1]), fk[slots], fv[slots], [10 ** 9], 0.1, 2 * 10 ** 9, 0)
        close(o[b:b + 1], want if n else (np.zeros(1), np.zeros(1)), f"row {b}, context {n}")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for step in range(4):
        g.replay()
        got = [x.clone() for x in out]
        torch.cuda.synchronize()
        for x, y in zip(got, call()):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), step
        for old, new in zip((cl, bt), contexts()):
            old.copy_(new)


def test_decode_more_sequences_than_a_split_holds():
    rng = np.random.default_rng(5)
    B, window = 8200, 20
    kc, vc = bf16(rng, 64, 16, 1, 64), bf16(rng, 64, 16, 1, 64)
    lens = rng.integers(0, 64, B)
    bt = torch.from_numpy(rng.integers(0, 64, (B, 4)).astype(np.int32)).to(DEV)
    q = bf16(rng, B, 2, 64)
    o = K.paged_attention_decode(q, kc, vc, torch.from_numpy(lens).to(DEV), bt, window=window, sinks=2)
    for b in list(range(0, B, 371)) + [8191, 8192, B - 1]:
        n = int(lens[b])
        k, v = (c[bt[b].long()].reshape(64, 1, 64)[:n] for c in (kc, vc))
        want = P.window_attention(f64(q[b:b + 1]), f64(k), f64(v), [n - 1], 0.125, window, 2) if n else (0.0, 0.0)
        close(o[b:b + 1], (np.zeros(1), np.zeros(1)) if n == 0 else want, f"row {b}")


def test_decode_bad_blocks_contribute_nothing_and_tables_end_the_context():
    """Entries outside the pool inside the window are skipped, as without a
    window; a context longer than its table ends there, the query staying at
    its place."""
    rng = np.random.default_rng(8)
    kc, vc, bt, seqs = paged(rng, [200, 200], [0, 0], 16, 2, 64, 0)
    q = bf16(rng, 2, 4, 64)
    bt[0, 11] = 10 ** 6
    bt[1, 10] = -1
    o = K.paged_attention_decode(q, kc, vc, torch.tensor([200, 200], device=DEV), bt, window=60)
    for b, gone in ((0, 11), (1, 10)):
        keep = np.r_[140:16 * gone, 16 * gone + 16:200] if gone > 8 else None
        keep = keep[keep >= 140]
        k, v = (x[keep] for x in seqs[b])
        close(o[b:b + 1], P.window_attention(f64(q[b:b + 1]), k, v, [len(keep)], 0.125, 1000, 0), f"row {b}")
    o = K.paged_attention_decode(q, kc, vc, torch.tensor([230, 200], device=DEV), bt[:, :12].contiguous(), window=60, sinks=3)
    k, v = seqs[0]
    keep = np.r_[0:3, 170:176]  # block 11 is outside the pool
    close(o[:1], P.window_attention(f64(q[:1]), k[keep], v[keep], [100], 0.125, 1000, 0), "longer than its table")


def test_windowed_calls_in_a_graph_and_on_another_stream():
    """Captured with new lengths, tables and keys between replays, every replay
    equal to the eager call; and a call on a side stream."""
    rng = np.random.default_rng(21)
    B, Hq, Hkv, D, window, sinks = 5, 8, 2, 64, 90, 4
    q, kc, vc = bf16(rng, B, Hq, D), bf16(rng, 40, 16, Hkv, D), bf16(rng, 40, 16, Hkv, D)
    bt = torch.from_numpy(rng.integers(0, 40, (B, 30)).astype(np.int32)).to(DEV)
    cl = torch.tensor([0, 5, 470, 91, 300], device=DEV)
    lens = [5, 60, 1]
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=DEV)
    pq, pk, pv = bf16(rng, 66, Hq, D), bf16(rng, 66, Hkv, D), bf16(rng, 66, Hkv, D)
    ws = torch.empty(max(16, K.paged_decode_window_workspace_bytes(B, Hq, D)), dtype=torch.uint8, device=DEV)

    def call():
        return (K.paged_attention_decode(q, kc, vc, cl, bt, workspace=ws, window=window, sinks=sinks),
                K.flash_attn_varlen_func(pq, pk, pv, cu, cu, 60, 60, window=33, sinks=2))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = call()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(on_side, call()):
        assert torch.equal(a, b)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for step in range(4):
        g.replay()
        got = [x.clone() for x in out]
        torch.cuda.synchronize()
        for a, b in zip(got, call()):
            assert torch.equal(a, b), step
        q.copy_(bf16(rng, B, Hq, D))
        pk.copy_(bf16(rng, 66, Hkv, D))
        cl.copy_(torch.from_numpy(rng.integers(0, 480, B)).to(DEV))
        bt.copy_(torch.from_numpy(rng.integers(0, 40, (B, 30)).astype(np.int32)).to(DEV))


def test_prefill_and_decode_agree_token_by_token():
    """A prompt's rows one at a time through the decode over the same keys."""
    rng = np.random.default_rng(31)
    n, Hq, Hkv, D, window, sinks, BS = 150, 8, 2, 64, 40, 3, 16
    q, k, v = bf16(rng, n, Hq, D), bf16(rng, n, Hkv, D), bf16(rng, n, Hkv, D)
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    a = K.flash_attn_varlen_func(q, k, v, cu, cu, n, n, window=window, sinks=sinks)
    kc, vc = (torch.zeros(10, BS, Hkv, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    K.store_kvcache(k, v, kc, vc, torch.arange(n, device=DEV))
    bt = torch.arange(10, dtype=torch.int32, device=DEV).expand(n, 10).contiguous()
    b = K.paged_attention_decode(q, kc, vc, torch.arange(1, n + 1, device=DEV), bt, window=window, sinks=sinks)
    for t in range(0, n, 7):
        want = P.window_attention(f64(q[t:t + 1]), f64(k), f64(v), [t], 0.125, window, sinks)
        close(a[t:t + 1], want, f"prefill {t}")
        close(b[t:t + 1], want, f"decode {t}")


def test_decode_pool_past_32_bit_offsets():
    """Blocks past element 2^31 of the pool (4 GiB of keys)."""
    rng = np.random.default_rng(41)
    NB, BS, Hkv, D = 33000, 256, 4, 64  # 2.16e9 elements
    kc = torch.zeros(NB, BS, Hkv, D, dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros_like(kc)
    lens, window, sinks = [900, 300], 400, 5
    bt = torch.full((2, 4), -1, dtype=torch.int32, device=DEV)
    ids = [32990, 32995, 32999, 32800, 32801, 32802]
    bt[0] = torch.tensor(ids[:4], dtype=torch.int32)
    bt[1, :2] = torch.tensor(ids[4:], dtype=torch.int32)
    q = bf16(rng, 2, 8, D)
    for b, n in enumerate(lens):
        k, v = bf16(rng, n, Hkv, D), bf16(rng, n, Hkv, D)
        t = torch.arange(n, device=DEV)
        slots = bt[b].long()[t // BS] * BS + t % BS
        K.store_kvcache(k, v, kc, vc, slots)
        cl = torch.tensor([n], device=DEV)
        want = P.window_attention(f64(q[b:b + 1]), f64(k), f64(v), [n - 1], 0.125, window, sinks)
        close(K.paged_attention_decode(q[b:b + 1], kc, vc, cl, bt[b:b + 1], window=window, sinks=sinks), want, f"{n}")
        cu = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
        ck = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        close(K.flash_attn_varlen_func(q[b:b + 1], kc, vc, cu, ck, 1, n, block_table=bt[b:b + 1], window=window,
                                       sinks=sinks), want, f"prefill {n}")


def test_refusals():
    rng = np.random.default_rng(1)
    q, kc = bf16(rng, 2, 4, 64), bf16(rng, 8, 16, 2, 64)
    cl, bt = torch.tensor([3, 4], device=DEV), torch.zeros(2, 1, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 2], dtype=torch.int32, device=DEV)
    k3 = bf16(rng, 2, 2, 64)
    for bad in (dict(window=0), dict(window=-3), dict(window=4, sinks=-1), dict(sinks=2)):
        with pytest.raises(ValueError):
            K.paged_attention_decode(q, kc, kc, cl, bt, **bad)
        with pytest.raises(ValueError):
            K.flash_attn_varlen_func(q, k3, k3, cu, cu, 2, 2, **bad)
    with pytest.raises(AssertionError, match="blocks_per_split"):
        K.paged_attention_decode(q, kc, kc, cl, bt, window=4, blocks_per_split=1)
    with pytest.raises(TypeError):
        K.paged_attention_decode(q.float(), kc, kc, cl, bt, window=4)
    with pytest.raises(ValueError, match="GPU only"):
        K.paged_attention_decode(q.cpu(), kc, kc, cl, bt, window=4)


def test_decode_tables_wider_than_any_window():
    """What counts against the balanced split is what is seen, not the table's
    width: 8192 rows of 32768 blocks, a few contexts of millions of tokens."""
    rng = np.random.default_rng(51)
    B, Hq, Hkv, D, BS, NB, width, window, sinks = 8192, 8, 8, 64, 256, 100, 32768, 4096, 4
    kc, vc, q = bf16(rng, NB, BS, Hkv, D), bf16(rng, NB, BS, Hkv, D), bf16(rng, B, Hq, D)
    lens = rng.integers(0, 300, B)
    far = {0: width * BS, 17: width * BS - 1, 4000: 5000001, 8191: 70000}
    bt = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    bt[:, :2] = torch.from_numpy(rng.integers(0, NB, (B, 2)).astype(np.int32)).to(DEV)
    for b, n in far.items():
        lens[b] = n
        lo, hi = (n - window) // BS, -(-n // BS)
        bt[b, lo:hi] = torch.from_numpy(rng.integers(0, NB, hi - lo).astype(np.int32)).to(DEV)
    o = K.paged_attention_decode(q, kc, vc, torch.from_numpy(lens).to(DEV), bt, window=window, sinks=sinks)
    for b in list(far) + [1, 2, 3, 5000, 8190]:
        n = int(lens[b])
        t = np.r_[0:min(sinks, max(0, n - window)), max(0, n - window):n]
        ids = bt[b].cpu().numpy()[t // BS]
        k, v = (f64(c[torch.from_numpy(ids).long().to(DEV), torch.from_numpy(t % BS).to(DEV)]) for c in (kc, vc))
        want = P.window_attention(f64(q[b:b + 1]), k, v, [len(t)], 0.125, 10 ** 9, 0)
        close(o[b:b + 1], want if n else (np.zeros(1), np.zeros(1)), f"row {b}, context {n}")


@pytest.mark.parametrize("B,Hq,Hkv,D,BS,window,sinks", [(45, 12, 4, 64, 16, 810, 4), (47, 32, 8, 128, 16, 790, 33),
                                                       (70, 8, 8, 64, 16, 520, 0), (33, 8, 4, 64, 64, 4100, 70),
                                                       (45, 12, 4, 64, 16, 810, 1500)])
def test_decode_long_windows_over_freed_blocks(B, Hq, Hkv, D, BS, window, sinks):
    """The equal share of all visible tiles per workgroup as the engine runs it:
    blocks behind the window freed (-1), NaN in everything hidden; then with
    entries outside the pool among the visible ones, which are skipped."""
    rng = np.random.default_rng(B + sinks)
    lens = rng.integers(0, 3 * window, B)
    lens[:7] = 0, 1, window, window + 1, window + sinks, window + BS, 3 * window
    kc, vc, bt, seqs = paged(rng, lens.tolist(), (lens - window).tolist(), BS, Hkv, D, sinks)
    q = bf16(rng, B, Hq, D)
    cl = torch.from_numpy(lens).to(DEV)
    table = bt.cpu().numpy()
    assert (table[6] == -1).sum() > 5
    for bad in (False, True):
        if bad:
            seen = np.argwhere(table >= 0)
            gone = seen[rng.permutation(len(seen))[:len(seen) // 5]]
            table[gone[:, 0], gone[:, 1]] = np.where(np.arange(len(gone)) % 2, -1, len(kc) + 3)
            bt = torch.from_numpy(table).to(DEV)
        o, oq, os_ = K.paged_attention_decode(q, kc, vc, cl, bt, 0.1, quant=True, window=window, sinks=sinks)
        assert torch.equal(o, K.paged_attention_decode(q, kc, vc, cl, bt, 0.1, window=window, sinks=sinks))
        wq, ws = K.act_quant(o.view(B, -1))
        assert torch.equal(oq.view(torch.uint8), wq.view(torch.uint8)) and torch.equal(os_, ws)
        for b, (n, (k, v)) in enumerate(zip(lens.tolist(), seqs)):
            t = np.arange(n)
            ids = table[b][t // BS]
            t = t[((t >= n - window) | (t < sinks)) & (ids >= 0) & (ids < len(kc))]
            want = P.window_attention(f64(q[b:b + 1]), k[t], v[t], [len(t)], 0.1, 10 ** 9, 0) if len(t) else (np.zeros(1), np.zeros(1))
            close(o[b:b + 1], want, f"row {b}, context {n}")


@pytest.mark.parametrize("B,Hq,Hkv,D,BS,window,sinks", [(1, 12, 4, 64, 256, 64, 4096), (3, 32, 8, 128, 16, 17, 1000),
                                                       (2, 8, 8, 64, 48, 1, 333), (5, 8, 1, 128, 64, 1000, 2000),
                                                       (90, 12, 4, 64, 16, 40, 700)])
def test_many_sinks_before_a_short_window(B, Hq, Hkv, D, BS, window, sinks):
    """A long beginning that stays visible: contexts inside it, at its end and
    past it, in the decode and as a chunk of new tokens."""
    rng = np.random.default_rng(B + sinks)
    lens = rng.integers(1, 2 * sinks, B)
    lens[:4] = [sinks + window + 40, sinks, sinks + 1, sinks // 2][:min(B, 4)]
    new = np.minimum(lens, 70)
    kc, vc, bt, seqs = paged(rng, lens.tolist(), (lens - new - window + 1).tolist(), BS, Hkv, D, sinks)
    q = bf16(rng, B, Hq, D)
    o = K.paged_attention_decode(q, kc, vc, torch.from_numpy(lens).to(DEV), bt, window=window, sinks=sinks)
    cq, ck = (torch.from_numpy(np.concatenate([[0], np.cumsum(x)]).astype(np.int32)).to(DEV) for x in (new, lens))
    pq = bf16(rng, int(new.sum()), Hq, D)
    po = K.flash_attn_varlen_func(pq, kc, vc, cq, ck, int(new.max()), int(lens.max()), block_table=bt, window=window,
                                  sinks=sinks)
    at = 0
    for b, (n, m, (k, v)) in enumerate(zip(lens.tolist(), new.tolist(), seqs)):
        close(o[b:b + 1], P.window_attention(f64(q[b:b + 1]), k, v, [n - 1], D ** -0.5, window, sinks), f"context {n}")
        if b < 8:
            close(po[at:at + m], P.window_attention(f64(pq[at:at + m]), k, v, np.arange(n - m, n), D ** -0.5, window,
                                                    sinks), f"{m} new of {n}")
        at += m
