"""qk_head_norm_rope_store (HIP) against float64.

Tolerance: one rounding to bf16 (half a step, 2^-8 of the value) and fp32
arithmetic: a norm of 128 squares, its rsqrt and four products come to less
than 2^-18 of |y1| + |y2|, the two values a rotated one is made of."""
import numpy as np
import pytest
import torch

from llm_from_scratch_amd import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 1e-6


def inputs(T, Hq, Hkv, D, R, seed, pad=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    full = torch.randn(T, (Hq + 2 * Hkv) * D + pad, generator=g, device=DEV).mul(scale).to(torch.bfloat16)
    ang = torch.outer(torch.arange(500, device=DEV).double(), 10000.0 ** (-torch.arange(0, R, 2, device=DEV).double() / R))
    return dict(qkv=full[:, :(Hq + 2 * Hkv) * D], q_weight=torch.randn(D, generator=g, device=DEV),
                k_weight=torch.randn(D, generator=g, device=DEV), cos_sin=torch.cat([ang.cos(), ang.sin()], -1).float(),
                positions=torch.randint(0, 500, (T,), generator=g, device=DEV), num_q_heads=Hq, num_kv_heads=Hkv, eps=EPS)


def check(got, x, weight, a, what):
    """x [T, H, D] in, got out."""
    x, w, cs = x.double(), weight.double(), a["cos_sin"].double()
    R = cs.shape[1]
    p = a["positions"].clamp(0, cs.shape[0] - 1)
    c, s = cs[p, None, :R // 2], cs[p, None, R // 2:]
    y = x / (x.square().mean(-1, keepdim=True) + a["eps"]).sqrt() * w
    lo, hi = y[..., :R // 2], y[..., R // 2:R]
    want = torch.cat([lo * c - hi * s, hi * c + lo * s, y[..., R:]], -1)
    size = torch.cat([lo.abs() + hi.abs()] * 2 + [y[..., R:].abs()], -1)
    err = (got.double() - want).abs()
    tol = 2.0 ** -8 * want.abs() + 2.0 ** -18 * size + 1e-38
    assert (err <= tol).all(), (what, (err / tol).max().item())


@pytest.mark.parametrize("Hq,Hkv,D,R", [(12, 4, 64, 64), (32, 8, 128, 128), (32, 8, 128, 64), (8, 8, 64, 16), (15, 3, 64, 32),
                                        (1, 1, 128, 112), (14, 2, 128, 32), (64, 8, 128, 128)])
@pytest.mark.parametrize("T", [1, 5, 700])
def test_values_and_slots(Hq, Hkv, D, R, T):
    a = inputs(T, Hq, Hkv, D, R, seed=T + Hq, pad=8)
    NB, BS = T // 16 + 3, 16
    kc, vc = (torch.full((NB, BS, Hkv, D), 7.0, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    slots = torch.randperm(NB * BS, device=DEV)[:T]
    slots[::4] = -1
    slots[1::7] = NB * BS + 5  # outside: skipped too
    q, k, v = K.qk_head_norm_rope_store(**a, k_cache=kc, v_cache=vc, slot_mapping=slots, return_kv=True)
    x = a["qkv"].reshape(T, Hq + 2 * Hkv, D)
    check(q, x[:, :Hq], a["q_weight"], a, "q")
    check(k, x[:, Hq:Hq + Hkv], a["k_weight"], a, "k")
    assert torch.equal(v, x[:, Hq + Hkv:])
    want_k, want_v = torch.full_like(kc, 7.0).view(-1, Hkv, D), torch.full_like(vc, 7.0).view(-1, Hkv, D)
    ok = (slots >= 0) & (slots < NB * BS)
    want_k[slots[ok]], want_v[slots[ok]] = k[ok], v[ok]
    assert torch.equal(kc.view(-1, Hkv, D), want_k) and torch.equal(vc.view(-1, Hkv, D), want_v)
    # without token-order outputs, without slots: the same bits
    kc2, vc2 = torch.full_like(kc, 7.0), torch.full_like(vc, 7.0)
    assert torch.equal(K.qk_head_norm_rope_store(**a, k_cache=kc2, v_cache=vc2, slot_mapping=slots), q)
    assert torch.equal(kc2, kc) and torch.equal(vc2, vc)
    q3, k3, v3 = K.qk_head_norm_rope_store(**a, return_kv=True)
    assert torch.equal(q3, q) and torch.equal(k3, k) and torch.equal(v3, v)


@pytest.mark.parametrize("Hq,Hkv,D,R,T", [(12, 4, 64, 64, 2048), (32, 8, 128, 64, 2053), (15, 3, 64, 32, 3001),
                                          (1, 1, 128, 128, 2500), (5, 2, 64, 16, 20001)])
def test_many_tokens(Hq, Hkv, D, R, T):
    """A wave per token, also more tokens than the grid has waves."""
    test_values_and_slots(Hq, Hkv, D, R, T)


def test_extremes():
    """Zero heads stay 0 (eps), large ones keep their direction, positions
    outside the table read its ends, no token is no launch."""
    a = inputs(64, 4, 2, 64, 64, seed=9, scale=1e15)
    a["qkv"][3] = 0
    a["qkv"][5] *= 1e-30
    a["positions"][:4] = torch.tensor([-5, 10 ** 12, 499, 0], device=DEV)
    q, k, v = K.qk_head_norm_rope_store(**a, return_kv=True)
    x = a["qkv"].reshape(64, 8, 64)
    check(q, x[:, :4], a["q_weight"], a, "q")
    check(k, x[:, 4:6], a["k_weight"], a, "k")
    assert (q[3] == 0).all() and (v[3] == 0).all()
    empty = dict(a, qkv=a["qkv"][:0], positions=a["positions"][:0])
    assert K.qk_head_norm_rope_store(**empty).shape == (0, 4, 64)


def test_in_a_graph_and_on_another_stream():
    a = inputs(33, 12, 4, 64, 64, seed=4)
    kc, vc = (torch.zeros(4, 16, 4, 64, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    slots = torch.randperm(64, device=DEV)[:33]

    def call(kc, vc):
        return K.qk_head_norm_rope_store(**a, k_cache=kc, v_cache=vc, slot_mapping=slots)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = call(kc.clone(), vc.clone())
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(side, call(kc.clone(), vc.clone()))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call(kc, vc)
    for i in range(3):
        a["qkv"].copy_(torch.randn_like(a["qkv"]))
        a["positions"].copy_(torch.randint(0, 500, (33,), device=DEV))
        g.replay()
        k2, v2 = torch.zeros_like(kc), torch.zeros_like(vc)
        assert torch.equal(out, call(k2, v2)) and torch.equal(kc, k2) and torch.equal(vc, v2)


def test_refusals():
    a = inputs(4, 4, 2, 64, 64, seed=1)
    for change, err in ((dict(q_weight=a["q_weight"][:32].contiguous()), AssertionError),
                        (dict(cos_sin=a["cos_sin"][:, :24].contiguous()), ValueError),
                        (dict(cos_sin=torch.zeros(10, 128, device=DEV)), ValueError),
                        (dict(cos_sin=a["cos_sin"][:0]), ValueError),
                        (dict(qkv=a["qkv"].float()), TypeError),
                        (dict(num_q_heads=5), AssertionError),
                        (dict(slot_mapping=a["positions"]), AssertionError),
                        (dict(positions=a["positions"][:3]), AssertionError),
                        (dict(positions=a["positions"].int()), TypeError),
                        (dict(qkv=a["qkv"].cpu()), ValueError),
                        (dict(qkv=torch.zeros(4, 8 * 96, device=DEV, dtype=torch.bfloat16), q_weight=torch.zeros(96, device=DEV),
                              k_weight=torch.zeros(96, device=DEV)), ValueError)):
        with pytest.raises(err):
            K.qk_head_norm_rope_store(**dict(a, **change))
