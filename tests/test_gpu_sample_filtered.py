"""sample_filtered (HIP) against a float64 oracle: the same token for every
row (bf16 logits and fp32 u put no border within 1e-10 of a draw by design of
the cases but for exact ties, which both resolve to the lowest index), and the
log-probability to a rounding to fp32 (half a step, 2^-24) plus 1e-9."""
import numpy as np
import pytest
import torch

from llm_from_scratch_amd import kernels as K
from oracle import sampler as S

pytestmark = pytest.mark.gpu
DEV = "cuda"


def run(logits, T, u, k=None, p=None, m=None):
    """Kernel and oracle on one batch; the arguments are lists or arrays."""
    B = logits.shape[0]
    t = [None if x is None else torch.tensor(np.broadcast_to(np.asarray(x, d), B).copy(), device=DEV)
         for x, d in ((T, np.float32), (u, np.float32), (k, np.int32), (p, np.float32), (m, np.float32))]
    tok, lp = K.sample_filtered(logits, t[0], t[1], top_k=t[2], top_p=t[3], min_p=t[4], return_logprob=True)
    assert tok.dtype == torch.int64 and lp.dtype == torch.float32 and tok.shape == lp.shape == (B,)
    alone = K.sample_filtered(logits, t[0], t[1], top_k=t[2], top_p=t[3], min_p=t[4])
    assert torch.equal(alone, tok)
    host = [None if x is None else x.cpu().numpy() for x in t]
    rows, tok, lp = logits.double().cpu().numpy(), tok.cpu().numpy(), lp.double().cpu().numpy()
    for b in range(B):
        a = [float(host[0][b]), float(host[1][b])] + [d if x is None else x[b] for x, d in
                                                     ((host[2], 0), (host[3], 1.0), (host[4], 0.0))]
        want, wlp = S.sample_filtered(rows[b], a[0], a[1], int(a[2]), float(a[3]), float(a[4]))
        assert tok[b] == want, (b, tok[b], want, a)
        assert lp[b] == wlp or abs(lp[b] - wlp) <= 2.0 ** -24 * abs(wlp) + 1e-9, (b, lp[b], wlp)


def logits_of(B, V, spread, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(B, V, generator=g, device=DEV) * spread).to(torch.bfloat16)


@pytest.mark.parametrize("B,V", [(1, 1), (2, 2), (3, 7), (5, 64), (4, 1001), (16, 32000), (3, 65536), (8, 150001), (2, 300000)])
@pytest.mark.parametrize("filters", ["", "k", "p", "m", "kpm"])
def test_tokens(B, V, filters):
    rng = np.random.default_rng(V + len(filters))
    for spread in (0.3, 2.5, 12.0):
        run(logits_of(B, V, spread, V), rng.uniform(0.4, 1.5, B), rng.random(B, np.float32),
            rng.choice([0, 1, 2, 40, 1000, V, V + 5, -3], B) if "k" in filters else None,
            rng.choice([0.0, 0.1, 0.5, 0.9, 0.999, 1.0, 1.5], B) if "p" in filters else None,
            rng.choice([0.0, 1e-6, 0.01, 0.5, 1.0, 2.0, -1.0], B) if "m" in filters else None)


@pytest.mark.parametrize("spread", [1e-30, 1e-3, 1.0, 1e30])
def test_min_p_cuts_anywhere(spread):
    """The last token that reaches min-p beside the largest, far from it, and
    next to 0, where neighbouring logits lie closer than 32 bits resolve the
    cut; over all chunks of values, of both signs and none."""
    B, V = 48, 3000
    logits = logits_of(B, V, spread, 31)
    logits[:, ::5] *= 1e-4
    logits[40:, 1:] = -logits[40:, 1:].abs()
    logits[44:, 0] = -0.0
    T = np.full(B, spread, np.float32)
    top = logits.double().amax(1).cpu().numpy() / T
    rng = np.random.default_rng(8)
    near = np.minimum(np.exp(-top * (1 + np.where(np.arange(B) % 3 == 0, 0, 1e-3) * rng.standard_normal(B))), 1.0)
    run(logits, T, rng.random(B, np.float32), m=np.where(np.arange(B) % 4 == 1, rng.random(B), near))
    run(logits, T, rng.random(B, np.float32), k=2000, p=0.99, m=near)


def test_equal_logits():
    """Every cut falls inside one bin: also with more equal logits than 16 bits
    count, where the token is floor(u n)."""
    for V in (10, 1000, 65535, 65536, 65537, 140000):
        for value in (0.0, -3.0, 88.0, 3e38, -3e38):
            logits = torch.full((6, V), value, device=DEV, dtype=torch.bfloat16)
            u = np.array([0, 0.25, 0.5, 0.999, 1 - 2.0 ** -24, 0.75], np.float32)
            run(logits, 0.7, u)
            run(logits, 0.7, u, k=[0, 3, 1, V // 2, 5, V], p=[1, 1, 0.5, 0.5, 0.3, 0.25], m=[1.0, 0, 0, 0, 1, 0.5])


def test_two_values_and_signed_zeros():
    """-0 and +0 are equal: the lower index comes first."""
    V = 5000
    logits = torch.zeros(4, V, device=DEV, dtype=torch.bfloat16)
    logits[:, ::2] = -0.0
    logits[1, 4000] = 1.0
    logits[2, 100:200] = -1.0
    run(logits, 1.0, [0.3, 0.9, 0.97, 0.0])
    run(logits, 1.0, [0.3, 0.9, 0.97, 0.0], k=[10, 10, 4901, 1], p=0.5)


def test_masked_rows():
    """-infinity, the type's lowest value, NaN and +infinity among the logits."""
    V = 40000
    low = torch.finfo(torch.bfloat16).min
    logits = logits_of(9, V, 2.0, 77)
    logits[0, 5:] = float("-inf")
    logits[1, :] = float("-inf")
    logits[2, :] = float("-inf")
    logits[2, 31234] = -2.0
    logits[3, 100:] = low
    logits[4, :] = low
    logits[5, ::3] = float("nan")
    logits[6, :] = float("nan")
    logits[7, [7, 9, 30000]] = float("inf")
    logits[8, :] = low
    logits[8, 17] = 3e38
    u = np.array([0.3, 0.4, 0.99, 0.999999, 0.5, 0.2, 0.1, 0.7, 0.9], np.float32)
    run(logits, 0.8, u)
    run(logits, 0.8, u, k=50, p=0.9, m=0.001)
    run(logits, 0.8, u, k=39999)


def test_temperatures_and_numbers_outside():
    """T <= 0 and NaN take the largest logit, tiny ones too; huge ones are
    uniform; u outside [0, 1) counts as the nearest inside, NaN as 0."""
    logits = logits_of(8, 3000, 3.0, 5)
    logits[:, [11, 900]] = 30.0
    run(logits, [0.0, -1.0, float("nan"), 1e-30, 1e-3, 1e30, float("inf"), 100.0], 0.9)
    t = torch.ones(4, device=DEV)
    got = K.sample_filtered(logits[:4], t, torch.tensor([-0.5, float("nan"), 1.0, 7.0], device=DEV))
    last = np.nextafter(np.float32(1), np.float32(0))
    want = K.sample_filtered(logits[:4], t, torch.tensor([0, 0, last, last], device=DEV))
    assert torch.equal(got, want)
    nan = torch.full((4,), float("nan"), device=DEV)
    u = torch.rand(4, device=DEV)
    assert torch.equal(K.sample_filtered(logits[:4], t, u, top_p=nan, min_p=nan), K.sample_filtered(logits[:4], t, u))


def test_strides_and_broadcast_rows():
    rng = np.random.default_rng(3)
    big = logits_of(10, 4100, 2.0, 3)
    for view in (big[:, 1:4000], big[::2, :4097], big[:5, 3:], big[2:3].expand(7, 4100)):
        run(view, rng.uniform(0.5, 1, view.shape[0]), rng.random(view.shape[0], np.float32), p=0.95)


def test_settings_of_any_stride():
    x, B = logits_of(6, 900, 2.0, 9), 6
    g = torch.Generator(device=DEV).manual_seed(2)
    u = torch.rand(2 * B, generator=g, device=DEV)[::2]
    t, p = torch.full((1,), 0.7, device=DEV).expand(B), torch.full((1,), 0.9, device=DEV).expand(B)
    assert torch.equal(K.sample_filtered(x, t, u, top_p=p),
                       K.sample_filtered(x, t.contiguous(), u.contiguous(), top_p=p.contiguous()))


def test_frequencies():
    logits = torch.tensor([[0.0, 1.0, 2.0, -1.0, 0.5]], device=DEV).to(torch.bfloat16)
    n = 40000
    g = torch.Generator(device=DEV).manual_seed(1)
    tok = K.sample_filtered(logits.expand(n, 5), torch.full((n,), 0.7, device=DEV), torch.rand(n, generator=g, device=DEV),
                            top_k=torch.full((n,), 3, device=DEV, dtype=torch.int32))
    p = torch.softmax(logits[0, [1, 2, 4]].float() / 0.7, 0).cpu().numpy()
    freq = np.bincount(tok.cpu().numpy(), minlength=5) / n
    # five standard deviations of a share of 40000 draws are under 0.0125
    assert freq[0] == freq[3] == 0 and np.abs(freq[[1, 2, 4]] - p).max() < 0.0125


def test_in_a_graph_and_on_another_stream():
    B, V = 6, 33000
    logits, t, u = logits_of(B, V, 2.0, 1), torch.rand(B, device=DEV) + 0.5, torch.rand(B, device=DEV)
    p = torch.full((B,), 0.95, device=DEV)

    def call():
        return K.sample_filtered(logits, t, u, top_p=p, return_logprob=True)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = call()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(side, call()))
    g, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    with torch.cuda.graph(g2, g.pool()):
        out2 = call()
    for i in range(4):
        logits.copy_(logits_of(B, V, 1.0 + i, i))
        u.copy_(torch.rand(B, device=DEV))
        (g if i % 2 else g2).replay()
        got = [x.clone() for x in (out if i % 2 else out2)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, call())), i


def test_no_rows_and_refusals():
    x, one = logits_of(2, 100, 1.0, 1), torch.ones(2, device=DEV)
    assert K.sample_filtered(x[:0], one[:0], one[:0]).shape == (0,)
    for args, kw, err in (((x.float(), one, one), {}, TypeError), ((x, one.double(), one), {}, TypeError),
                          ((x, one, one), dict(top_k=torch.ones(2, device=DEV, dtype=torch.int64)), TypeError),
                          ((x, one, one[:1]), {}, AssertionError), ((x, one, one), dict(top_p=one[:1]), AssertionError),
                          ((x.t(), one, one), {}, AssertionError), ((x.cpu(), one, one), {}, ValueError),
                          ((x, one, one), dict(min_p=one.cpu()), ValueError), ((x[:, :0], one, one), {}, ValueError)):
        with pytest.raises(err):
            K.sample_filtered(*args, **kw)


@pytest.mark.parametrize("filters", ["", "k", "p", "m", "kpm"])
def test_several_values_past_16_bit_counts(filters):
    """Rows in which a value that is not the shared one has more tokens than 16
    bits count: above the others and below, of either sign, both signs of one
    value (the halves of one word), -0 beside +0, values that are never drawn.
    (p and the values put no border on a token: p n and m / w are no whole
    numbers and no ratios of weights.)"""
    rng = np.random.default_rng(61)
    inf, low = float("inf"), float(torch.finfo(torch.bfloat16).min)
    rows = [  # (value, tokens); the rest of a row is random
        [(3.0, 75000), (1.5, 75001)], [(-2.0, 75000), (-2.5, 75001)], [(2.0, 75001), (-2.0, 75000)],
        [(0.0, 75000), (-0.0, 75001)], [(-0.0, 75001), (0.0, 75000)], [(1.0, 70000), (0.5, 70000)],
        [(float("nan"), 70000), (0.25, 70000)], [(-inf, 70000), (-1.0, 70000)], [(low, 70000), (2.0, 70000)],
        [(2.0, 70000), (low, 70000)], [(88.0, 66000), (87.5, 65537)], [(inf, 70000), (5.0, 70000)]]
    wide = [[(0.75, 90000), (1.25, 66000), (-1.25, 66000)], [(-3.0, 90000), (-0.5, 66000), (0.5, 70000)],
            [(4.0, 90000), (0.0, 66000), (-0.0, 66000)], [(-inf, 90000), (float("nan"), 66000), (-1.0, 70000)]]
    for V, batch in ((150001, rows), (230003, wide)):
        x = rng.standard_normal((len(batch), V)).astype(np.float32)
        for b, values in enumerate(batch):
            # the first value's tokens at the front too, where the samples' first lanes find it
            at, first = np.r_[np.arange(9000), 9000 + rng.permutation(V - 9000)], 0
            for value, n in values:
                x[b, at[first:first + n]] = value
                first += n
        logits = torch.from_numpy(x).to(DEV).to(torch.bfloat16)
        B = len(batch)
        run(logits, rng.uniform(0.6, 1.4, B), rng.random(B, np.float32),
            rng.choice([1, 7001, 70011, 80001, 140001], B) if "k" in filters else None,
            rng.choice([0.137, 0.533, 0.911, 0.9993], B) if "p" in filters else None,
            rng.choice([1e-5, 0.013, 0.77], B) if "m" in filters else None)
