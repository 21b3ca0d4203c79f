"""Without a GPU: the oracle of the logit penalties against a brute force, and
the host-side checks of the operators' C entries (nothing is launched)."""
import numpy as np
import pytest

from llm_from_scratch_amd import _lib
from oracle import sampler as S


def test_penalties_oracle():
    rng = np.random.default_rng(0)
    for _ in range(200):
        V = int(rng.integers(1, 9))
        x = rng.normal(0, 2, V)
        history = rng.integers(-1, V + 1, int(rng.integers(0, 12))).tolist()
        np_, r, p, f = int(rng.integers(0, 14)), rng.uniform(0.5, 2), rng.normal(), rng.normal()
        pairs = [(int(rng.integers(-1, V + 1)), rng.normal()) for _ in range(int(rng.integers(0, 4)))]
        ok = rng.random(V) < 0.7
        want = []
        for v in range(V):
            y = x[v]
            if v in history:
                y = y / r if y > 0 else y * r
            c = sum(1 for i, t in enumerate(history) if t == v and i >= np_)
            y = y - f * c - (p if c else 0.0) + sum(b for t, b in pairs if t == v)
            want.append(y if ok[v] else -np.inf)
        np.testing.assert_allclose(S.apply_penalties(x, history, np_, r, p, f, pairs, ok), want, atol=1e-12)


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def refused(lib, rc, why):
    assert rc == -1 and why in lib.lfs_last_error(), (rc, lib.lfs_last_error())


def test_store_and_load_refusals(lib):
    def store(T=4, Hkv=4, D=64, BS=16, NB=8, key=16, kc=16, ks=16, slots=16):
        return lib.lfs_store_kvcache_fp8(key, Hkv * D, 16, Hkv * D, kc, 16, ks, 16, slots, T, Hkv, D, BS, NB, None)

    refused(lib, store(D=96), b"head_dim")
    refused(lib, store(T=-1), b"bad shape")
    refused(lib, store(BS=0), b"bad shape")
    refused(lib, store(key=None), b"null pointer")
    refused(lib, store(ks=None), b"null pointer")
    refused(lib, store(kc=20), b"8-byte aligned")
    refused(lib, store(T=1 << 29), b"too many tokens")
    assert store(T=0, key=None, slots=None) == 0

    def load(B=2, total=8, Hkv=4, D=64, BS=16, NB=8, bts=4, mb=4, cu=16, kc=16, bt=16, k=16):
        return lib.lfs_load_kvcache_fp8(kc, 16, 16, 16, bt, bts, mb, cu, B, total, k, 16, Hkv, D, BS, NB, None)

    refused(lib, load(D=32), b"head_dim")
    refused(lib, load(B=-1), b"bad shape")
    refused(lib, load(total=-1), b"bad shape")
    refused(lib, load(bts=3), b"stride")
    refused(lib, load(cu=None), b"null pointer")
    refused(lib, load(bt=None), b"null block table")
    refused(lib, load(kc=8), b"16-byte aligned")
    refused(lib, load(k=24), b"16-byte aligned")
    refused(lib, load(total=1 << 30), b"too many rows")
    assert load(total=0, cu=None, k=None) == 0


@pytest.mark.parametrize("shared", [False, True])
def test_decode_refusals(lib, shared):
    def call(B=2, Hq=8, Hkv=4, D=64, BS=16, NB=8, mb=4, bts=4, q=16, bt=16, ws=16, need=None, qo=None, qs=None, NG=1,
             cu=16, ks=16):
        if need is None:
            need = lib.lfs_paged_decode_shared_workspace_bytes(max(B, 0), max(NG, 0), Hq, Hkv, D) if shared else \
                lib.lfs_paged_decode_fp8_workspace_bytes(max(B, 0), Hq, D)
        tail = (16, ws, need, B, Hq, Hkv, D, BS, NB, mb, 0.1, qo, qs, None)
        if shared:
            return lib.lfs_paged_decode_shared(q, 16, 16, 16, bt, bts, cu, 16, NG, *tail)
        return lib.lfs_paged_decode_fp8(q, 16, 16, ks, 16, 16, bt, bts, *tail)

    refused(lib, call(D=96), b"head_dim")
    refused(lib, call(Hq=9, Hkv=1), b"ratio")
    refused(lib, call(BS=24), b"multiple of 16")
    refused(lib, call(bts=3), b"stride")
    refused(lib, call(NB=0), b"empty KV pool")
    refused(lib, call(q=None), b"null pointer")
    refused(lib, call(q=8), b"16-byte aligned")
    refused(lib, call(bt=None), b"null block table")
    refused(lib, call(B=65536), b"too large")
    refused(lib, call(need=16), b"workspace of 16 bytes")
    refused(lib, call(ws=None), b"workspace of")
    refused(lib, call(ws=8), b"workspace must be 16-byte aligned")
    refused(lib, call(qo=16), b"go together")
    refused(lib, call(Hq=1, Hkv=1, qo=16, qs=16), b"128")
    if shared:
        refused(lib, call(NG=-1), b"bad shape")
        refused(lib, call(cu=None), b"null pointer")
        refused(lib, call(B=8193), b"8192")
        refused(lib, call(NG=8193), b"8192")
    else:
        refused(lib, call(ks=None), b"null pointer")
        refused(lib, call(ks=8), b"scales must be 16-byte aligned")
    assert call(B=0, q=None) == 0


def test_penalty_refusals(lib):
    def call(B=2, V=100, ldo=100, tokens=16, width=5, pl=16, sl=16, rep=16, ids=None, bias=None, n=0, allowed=None, mst=4,
             x=16):
        return lib.lfs_apply_penalties(x, 100, 16, ldo, 0, tokens, 5, width, pl, sl, rep, None, None, ids, bias, n, allowed,
                                       mst, B, V, None)

    refused(lib, call(B=-1), b"bad shape")
    refused(lib, call(B=65536), b"bad shape")
    refused(lib, call(V=1 << 30), b"bad shape")
    refused(lib, call(x=None), b"null pointer")
    refused(lib, call(ldo=99), b"overlap")
    refused(lib, call(sl=None), b"go together")
    refused(lib, call(tokens=None), b"go together")
    refused(lib, call(tokens=None, pl=None, sl=None), b"need the rows' tokens")
    refused(lib, call(n=2), b"go together")
    refused(lib, call(n=1025, ids=16, bias=16), b"1024")
    refused(lib, call(allowed=16, mst=3), b"too few words")
    assert call(B=0, x=None) == 0


def test_calls_past_the_threads_of_a_launch_are_refused(lib):
    """2^32 threads: the host's error, not the launch's."""
    for T, Hkv in ((1 << 28, 1), ((1 << 28) - 15, 2)):
        refused(lib, lib.lfs_load_kvcache_fp8(16, 16, 16, 16, 16, 4, 4, 16, 1, T, 16, 16, Hkv, 64, 16, 8, None), b"too many rows")
    refused(lib, lib.lfs_store_kvcache_fp8(16, 64, 16, 64, 16, 16, 16, 16, 16, 1 << 28, 1, 64, 16, 8, None),
            b"too many tokens")
    B, Hq, Hkv, D = 8192, 8192, 1024, 64
    need = lib.lfs_paged_decode_shared_workspace_bytes(B, 1, Hq, Hkv, D)
    refused(lib, lib.lfs_paged_decode_shared(16, 16, 16, 16, 16, 4, 16, 16, 1, 16, 16, need, B, Hq, Hkv, D, 16, 8, 4, 0.1,
                                             None, None, None), b"too many outputs")
