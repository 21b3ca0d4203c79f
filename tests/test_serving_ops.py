"""Without a GPU: the oracles of windowed attention and filtered sampling
against brute force, and the host-side checks of the operators' C entries
(nothing is launched)."""
import ctypes
import math

import numpy as np
import pytest

from llm_from_scratch_amd import _lib
from llm_from_scratch_amd import kernels as K
from oracle import paged_kv as P
from oracle import sampler as S


@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 1), (2, 5), (100, 0)])
def test_window_oracle(window, sinks):
    rng = np.random.default_rng(window)
    q, k, v = rng.standard_normal((5, 2, 4)), rng.standard_normal((7, 1, 4)), rng.standard_normal((7, 1, 4))
    o, a = P.window_attention(q, k, v, [-1, 0, 3, 5, 6], 0.3, window, sinks)
    for i, p in enumerate([-1, 0, 3, 5, 6]):
        seen = [j for j in range(7) if j <= p and (j > p - window or j < sinks)]
        for h in range(2):
            w = [math.exp(0.3 * float(q[i, h] @ k[j, 0])) for j in seen]
            want = sum((x * v[j, 0] for x, j in zip(w, seen)), np.zeros(4)) / (sum(w) or 1)
            np.testing.assert_allclose(o[i, h], want, atol=1e-12)
    # values nobody sees take no part (the sums of another number of keys run in another order)
    v2 = v.copy()
    v2[~P.window_mask([6], 7, window, sinks)[0]] = np.nan
    np.testing.assert_allclose(P.window_attention(q[4:], k, v2, [6], 0.3, window, sinks)[0], o[4:], atol=1e-12)


def test_sampling_oracle():
    rng = np.random.default_rng(0)
    for _ in range(200):
        n = int(rng.integers(1, 9))
        x = rng.integers(-3, 4, n) / 2.0
        T, u, k, p, m = rng.uniform(0.3, 2), rng.random(), int(rng.integers(0, n + 2)), rng.choice([0.3, 0.8, 1.0]), \
            rng.choice([0.0, 0.2, 1.0])
        order = sorted(range(n), key=lambda i: (-x[i], i))
        w = {i: math.exp((x[i] - max(x)) / T) for i in order}
        kept = order[:k] if k > 0 else order
        if p < 1:
            total, cut = sum(w[i] for i in kept), []
            while not cut or sum(w[i] for i in cut) < p * total * (1 - 1e-12):
                cut.append(kept[len(cut)])
            kept = cut
        kept = [i for j, i in enumerate(kept) if j == 0 or w[i] >= m]
        total, at, tok = sum(w[i] for i in kept), 0.0, kept[-1]
        for i in kept:
            at += w[i]
            if at > u * total:
                tok = i
                break
        got, lp = S.sample_filtered(x, T, u, k, p, m)
        assert got == tok and lp == pytest.approx(math.log(w[tok] / total), abs=1e-12)
    assert S.sample_filtered([-np.inf, np.nan], 1.0, 0.5) == (0, -np.inf)
    assert S.sample_filtered([1.0, 3.0, 3.0], 0.0, 0.9) == (1, 0.0)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def refused(lib, rc, why):
    assert rc == -1 and why in lib.lfs_last_error(), (rc, lib.lfs_last_error())


def test_window_refusals(lib):
    def prefill(B=2, Hq=8, Hkv=4, D=64, max_q=4, window=8, sinks=0, bt=None, bts=0, BS=0, q=16):
        return lib.lfs_prefill_attention_window(q, 16, 16, 16, 16, bt, bts, BS, 64, 16, B, Hq, Hkv, D, max_q, window, sinks,
                                                0.1, None)

    refused(lib, prefill(D=96), b"head_dim")
    refused(lib, prefill(Hq=9, Hkv=1), b"ratio")
    refused(lib, prefill(window=0), b"window must be >= 1")
    refused(lib, prefill(sinks=-1), b"sinks")
    refused(lib, prefill(bt=16, bts=4, BS=24), b"multiple of 16")
    refused(lib, prefill(q=None), b"null pointer")
    refused(lib, prefill(q=8), b"aligned")
    assert prefill(B=0) == 0 and prefill(max_q=0) == 0

    def decode(B=2, Hq=8, Hkv=4, D=64, BS=16, NB=8, mb=4, bts=4, window=8, sinks=0, q=16, ws=16, wsb=1 << 30, qo=None):
        return lib.lfs_paged_decode_window(q, 16, 16, 16, 16, bts, 16, ws, wsb, B, Hq, Hkv, D, BS, NB, mb, window, sinks,
                                           0.1, qo, None, None)

    refused(lib, decode(D=80), b"head_dim")
    refused(lib, decode(Hq=6), b"multiple of num_kv_heads")
    refused(lib, decode(BS=8), b"block_size")
    refused(lib, decode(window=-1), b"window must be >= 1")
    refused(lib, decode(bts=3), b"stride")
    refused(lib, decode(NB=0), b"empty KV pool")
    refused(lib, decode(q=None), b"null pointer")
    refused(lib, decode(qo=16), b"go together")
    refused(lib, decode(ws=8), b"workspace must be 16-byte aligned")
    assert decode(B=0) == 0
    assert lib.lfs_paged_decode_window_workspace_bytes(-1, 8, 64) == -1


def test_copy_refusals(lib):
    def copy(src, dst, planes=2, nb=10, block=64, pool=16):
        arr = [(ctypes.c_int32 * max(1, len(x)))(*x) for x in (src, dst)]
        return lib.lfs_copy_kv_blocks(pool, planes, nb, block, *(ctypes.addressof(x) for x in arr), len(src), None)

    refused(lib, copy([1], [2], block=40), b"16 bytes")
    refused(lib, copy([1, 10], [2, 3]), b"outside the pool")
    refused(lib, copy([1, 3], [2, -1]), b"outside the pool")
    refused(lib, copy([1, 3], [2, 2]), b"twice")
    refused(lib, copy([1, 2], [2, 3]), b"source and a destination")
    refused(lib, copy([1], [2], pool=8), b"aligned")
    refused(lib, copy([1], [2], pool=None), b"null pointer")
    refused(lib, copy(range(11), range(11)), b"pairs for 10 blocks")
    assert copy([], []) == 0 and copy([1], [2], planes=0) == 0


def test_head_norm_and_sampling_refusals(lib):
    def norm(ld=1024, R=64, T=4, Hq=8, Hkv=4, D=64, maxp=10, q=16, ko=None, slots=None):
        return lib.lfs_qk_head_norm_rope_store(q, ld, 16, 16, 16, R, 16, slots, 16, None, None, ko, None, T, Hq, Hkv, D, 64,
                                               maxp, 1e-6, None)

    refused(lib, norm(D=96, ld=4096), b"head_dim")
    refused(lib, norm(R=24), b"rotary_dim")
    refused(lib, norm(R=80), b"rotary_dim")
    refused(lib, norm(ld=1020), b"row stride")
    refused(lib, norm(maxp=0), b"empty rotation table")
    refused(lib, norm(q=None), b"null pointer")
    refused(lib, norm(ko=16), b"go together")
    refused(lib, norm(slots=16), b"null cache")
    refused(lib, norm(T=1 << 40), b"too many tokens")
    assert norm(T=0) == 0

    def sample(logits=16, ld=100, B=2, V=100, u=16):
        return lib.lfs_sample_filtered(logits, ld, 16, u, None, None, None, B, V, 16, None, None)

    refused(lib, sample(ld=99), b"bad shape")
    refused(lib, sample(V=0), b"bad shape")
    refused(lib, sample(u=None), b"null pointer")
    refused(lib, sample(B=1 << 40), b"too many rows")
    assert sample(B=0) == 0


def test_host_block_ids():
    assert K._block_ids(range(3), "src").tolist() == [0, 1, 2]
    assert K._block_ids(np.array([4, 5]), "src").tolist() == [4, 5]
    with pytest.raises(ValueError, match="outside"):
        K._block_ids([2 ** 40], "src")
    with pytest.raises(TypeError):
        K._block_ids([1.5], "src")
