"""apply_penalties (HIP) against a float64 oracle.

Tolerance, per logit: a rounding to the logits' type (half a step: 2^-8 of it for
bf16, 2^-24 for fp32) and the fp32 steps before it: each of the division or
product, frequency * count, the two differences and the n additions of biases
rounds by at most 2^-24 of the sizes that meet there, whose sum bounds them all.
Masked logits and infinities are equal."""
import numpy as np
import pytest
import torch

from llm_from_scratch_amd import kernels as K
from oracle import sampler as S

pytestmark = pytest.mark.gpu
DEV = "cuda"


def dev(x, dtype):
    return None if x is None else torch.from_numpy(np.ascontiguousarray(np.asarray(x, dtype))).to(DEV)


def words(allowed):
    """Truth values [B, V] as int32 words, bit v % 32 of word v // 32."""
    B, V = allowed.shape
    bits = np.zeros((B, -(-V // 32) * 32), np.uint8)
    bits[:, :V] = allowed
    return np.packbits(bits, axis=1, bitorder="little").view(np.int32)


def check(logits, tokens=None, prompts=None, lens=None, rep=None, pres=None, freq=None, ids=None, bias=None,
          allowed=None, **kw):
    B, V = logits.shape
    rows = logits.double().cpu().numpy()
    got = K.apply_penalties(logits, dev(tokens, np.int32), dev(prompts, np.int32), dev(lens, np.int32),
                            dev(rep, np.float32), dev(pres, np.float32), dev(freq, np.float32), dev(ids, np.int32),
                            dev(bias, np.float32), None if allowed is None else dev(words(allowed), np.int32), **kw)
    assert got.dtype == logits.dtype and got.shape == (B, V)
    half = 2.0 ** -8 if logits.dtype == torch.bfloat16 else 2.0 ** -24
    out = got.double().cpu().numpy()

    def one(x, b, default):
        return default if x is None else float(np.float32(x[b]))

    for b in range(B):
        n = 0 if lens is None else max(0, min(int(lens[b]), tokens.shape[1]))
        history = [] if lens is None else tokens[b, :n]
        pairs = [] if ids is None else [(int(i), float(np.float32(v))) for i, v in zip(ids[b], bias[b])]
        r, p, f = one(rep, b, None), one(pres, b, 0.0), one(freq, b, 0.0)
        want = S.apply_penalties(rows[b], history, 0 if lens is None else int(prompts[b]), r, p, f, pairs,
                                 None if allowed is None else allowed[b])
        size = np.abs(np.where(np.isfinite(rows[b]), rows[b], 0)) * max(1.0, r or 1.0, 1.0 / (r or 1.0))
        size += (abs(f) * n + abs(p)) * (n > 0)
        for i, v in pairs:
            if 0 <= i < V and np.isfinite(v):
                size[i] += abs(v)
        # past the halfway point above the type's largest value, 2^128 (1 - half), lies its infinity
        want = np.where(np.abs(want) >= 2.0 ** 128 * (1 - half / 2), np.copysign(np.inf, want), want)
        fine = np.isfinite(want)
        assert np.array_equal(out[b][~fine], want[~fine], equal_nan=True), b
        tol = half * np.abs(want) + (4 + len(pairs)) * 2.0 ** -24 * size + 1e-38
        with np.errstate(invalid="ignore"):
            bad = np.flatnonzero(~(np.abs(out[b] - want) <= tol) & fine)
        assert not len(bad), (b, bad[:5], out[b][bad[:5]], want[bad[:5]])
    return got


def logits_of(rng, B, V, dtype=torch.bfloat16, spread=3.0):
    return torch.from_numpy((spread * rng.standard_normal((B, V))).astype(np.float32)).to(dtype).to(DEV)


SHAPES = [(1, 1), (2, 7), (3, 64), (4, 1001), (1, 32000), (5, 4096), (2, 8193), (3, 150001)]


@pytest.mark.parametrize("B,V", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("what", ["r", "pf", "rpf", "b", "m", "bm", "rpfbm", ""])
def test_parts(B, V, dtype, what):
    rng = np.random.default_rng(B * V + len(what))
    L = 300
    lens = rng.integers(0, L + 1, B)
    lens[0] = L
    tokens = (V * rng.random((B, L)) ** 3).astype(int)  # a few often
    history = dict(tokens=tokens, prompts=rng.integers(0, L, B), lens=lens) if set(what) & set("rpf") else {}
    n = min(V, 40)
    check(logits_of(rng, B, V, dtype), **history,
          rep=rng.uniform(0.5, 2.0, B) if "r" in what else None,
          pres=rng.uniform(-1, 2, B) if "p" in what else None,
          freq=rng.uniform(-0.2, 1, B) if "f" in what else None,
          ids=np.stack([rng.choice(V, n, replace=False) for _ in range(B)]) if "b" in what else None,
          bias=rng.normal(0, 20, (B, n)) if "b" in what else None,
          allowed=rng.random((B, V)) < 0.3 if "m" in what else None)


@pytest.mark.parametrize("V", [50, 9000])
def test_histories(V):
    """Prompts longer than the history, none and negative; lengths of 0, 1, past
    the tokens and below 0; ids outside the vocabulary; one token throughout; a
    history of many thousands."""
    rng = np.random.default_rng(V)
    L = 20000
    tokens = rng.integers(-5, V + 5, (9, L))
    tokens[3] = 7
    tokens[4, ::2] = 2 ** 31 - 1
    tokens[5] = -2 ** 31
    tokens[6] = V - 1
    tokens[7] = V
    check(logits_of(rng, 9, V), tokens, np.array([0, 5, -3, 10, 30000, 0, L - 1, 0, 0]),
          np.array([0, 1, 50, L, 20, L, L, 3000, 2 * L]) * np.array([1, 1, 1, 1, 1, 1, 1, 1, 1]),
          rep=np.full(9, 1.3), pres=np.full(9, 0.4), freq=np.full(9, 0.01))
    check(logits_of(rng, 2, V), tokens[:2], np.array([0, 0]), np.array([-4, 0]), rep=[1.5, 1.5], pres=[1, 1], freq=[1, 1])
    check(logits_of(rng, 2, V), tokens[:2, :0], np.array([0, 0]), np.array([3, 0]), rep=[1.5, 1.5])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("L", [900, 17000])
def test_large_batches(dtype, L):
    """Large chunks, with counts of either width, biases and masks, rows at odd
    addresses."""
    rng = np.random.default_rng(L)
    B, V = 24, 90001
    tokens = (V * (rng.integers(0, 300, (B, L)) / 300) ** 3).astype(int)
    check(logits_of(rng, B, V, dtype), tokens, rng.integers(0, L, B), rng.integers(0, L + 1, B), rep=rng.uniform(0.5, 2, B),
          pres=rng.uniform(0, 2, B), freq=rng.uniform(0, 0.1, B), ids=rng.integers(0, V, (B, 30)),
          bias=rng.normal(0, 9, (B, 30)), allowed=rng.random((B, V)) < 0.6)


def test_prompt_tokens_are_repeated_but_not_counted():
    x = torch.tensor([[2.0, -2.0, 2.0, -2.0, 1.0]], device=DEV)
    got = K.apply_penalties(x, dev([[0, 1, 2, 3, 3]], np.int32), dev([2], np.int32), dev([5], np.int32),
                            dev([2.0], np.float32), dev([0.25], np.float32), dev([0.5], np.float32))
    assert got.tolist() == [[1.0, -4.0, 0.25, -5.25, 1.0]]


def test_biases_of_one_token_add_up_in_order():
    rng = np.random.default_rng(5)
    V, n = 5000, 1024
    ids = rng.integers(-2, 30, (2, n)) * 170
    ids[1, :] = 4999
    check(logits_of(rng, 2, V, torch.float32), ids=ids, bias=rng.normal(0, 3, (2, n)))
    x = torch.zeros(1, 4, device=DEV)
    got = K.apply_penalties(x, bias_ids=dev([[1, 1, 1, 2]], np.int32), bias=dev([[1e8, 1.0, -1e8, 0.5]], np.float32))
    assert got.tolist() == [[0.0, 0.0, 0.5, 0.0]]  # (1e8 + 1) - 1e8 in fp32
    got = K.apply_penalties(x, bias_ids=dev([[-1, 3]], np.int32), bias=dev([[5.0, -np.inf]], np.float32))
    assert got.tolist() == [[0.0, 0.0, 0.0, -np.inf]]


def test_infinities_and_masks():
    rng = np.random.default_rng(6)
    V = 4099
    x = logits_of(rng, 4, V)
    x[0, ::3], x[1, ::5], x[2, 1::2] = -np.inf, np.inf, float("nan")
    x[3] = torch.finfo(torch.bfloat16).min
    tokens = rng.integers(0, V, (4, 900))
    for allowed in (None, np.zeros((4, V), bool), rng.random((4, V)) < 0.5, np.ones((4, V), bool)):
        check(x, tokens, np.full(4, 100), np.full(4, 900), rep=np.full(4, 1.25), pres=np.full(4, 0.5),
              freq=np.full(4, 0.1), allowed=allowed)
    with_bias = np.full((4, 1), 3)
    check(x, ids=with_bias, bias=np.full((4, 1), 7.0), allowed=np.zeros((4, V), bool))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [64, 1001, 9001])
def test_layouts(dtype, V):
    """Rows with a stride and at odd addresses, rows that are one, tokens,
    masks and biases with strides; out of its own and in place, whose other
    values stay."""
    rng = np.random.default_rng(V)
    B, L = 5, 70
    history = dict(tokens=rng.integers(0, V, (B, L)), prompts=np.full(B, 9), lens=rng.integers(0, L, B))
    more = dict(rep=np.full(B, 1.2), pres=np.full(B, 0.5), freq=np.full(B, 0.1), ids=rng.integers(0, V, (B, 3)),
                bias=rng.normal(0, 3, (B, 3)), allowed=rng.random((B, V)) < 0.8)
    for at, pad in ((0, 0), (1, 3), (3, 5), (8, 8)):
        wide = logits_of(rng, B, at + V + pad, dtype)
        want = check(wide[:, at:at + V].clone(), **history, **more)
        assert torch.equal(check(wide[:, at:at + V], **history, **more), want)
        out = torch.full((B, V + 6), 5.0, dtype=dtype, device=DEV)
        got = K.apply_penalties(wide[:, at:at + V], out=out[:, 2:V + 2])
        assert got.data_ptr() == out[:, 2:].data_ptr() and torch.equal(got, wide[:, at:at + V])
        assert (out[:, :2] == 5).all() and (out[:, V + 2:] == 5).all()
        held = wide.clone()
        check(wide[:, at:at + V], **history, **more, out=held[:, at:at + V])
        assert torch.equal(held[:, at:at + V], want)
        assert torch.equal(held[:, :at], wide[:, :at]) and torch.equal(held[:, at + V:], wide[:, at + V:])
        tokens, bits = (torch.zeros(B, 2 * x.shape[1] + 1, dtype=torch.int32, device=DEV)
                        for x in (history["tokens"], words(more["allowed"])))
        tokens[:, 1:L + 1], bits[:, :-(-V // 32)] = dev(history["tokens"], np.int32), dev(words(more["allowed"]), np.int32)
        place = wide[:, at:at + V]
        got = K.apply_penalties(place, tokens[:, 1:L + 1], dev(history["prompts"], np.int32),
                                dev(history["lens"], np.int32), *(dev(more[n], np.float32) for n in ("rep", "pres", "freq")),
                                bias_ids=dev(np.repeat(more["ids"], 2, 1), np.int32)[:, ::2],
                                bias=dev(np.repeat(more["bias"], 2, 1), np.float32)[:, ::2],
                                allowed=bits[:, :-(-V // 32)], out=place)
        assert got.data_ptr() == place.data_ptr() and torch.equal(wide, held)
    one = logits_of(rng, 1, V, dtype)
    assert torch.equal(check(one.expand(B, V), **history, **more), check(one.repeat(B, 1), **history, **more))


@pytest.mark.parametrize("V", [1, 77, 9001])
def test_single_rows_of_any_stride(V):
    """One row whose stride is not its width: of a transposed column (1), of
    every third row (3 V); as logits, as out, as tokens and as a mask."""
    rng = np.random.default_rng(V)
    tokens = rng.integers(0, V, (1, 20))
    more = dict(prompts=np.full(1, 3), lens=np.full(1, 20), rep=np.full(1, 1.5), pres=np.full(1, 0.5),
                freq=np.full(1, 0.1), allowed=rng.random((1, V)) < 0.8)
    flat = logits_of(rng, 1, V).view(V)
    want = check(flat.view(1, V), tokens, **more)
    for stride in (1, 3 * V):
        one = flat.as_strided((1, V), (stride, 1))
        assert torch.equal(check(one, tokens, **more), want)
        out = torch.empty(V, dtype=flat.dtype, device=DEV).as_strided((1, V), (stride, 1))
        check(one, tokens, **more, out=out)
        assert torch.equal(out, want)
        bits = dev(words(more["allowed"]), np.int32)
        got = K.apply_penalties(
            one, dev(tokens, np.int32).as_strided((1, 20), (stride, 1)), dev(more["prompts"], np.int32),
            dev(more["lens"], np.int32), dev(more["rep"], np.float32), dev(more["pres"], np.float32),
            dev(more["freq"], np.float32), allowed=bits.as_strided(bits.shape, (stride, 1)))
        assert torch.equal(got, want)


def test_rows_past_32_bits():
    V, B = 150000, 15000
    x = torch.empty(B, V, dtype=torch.bfloat16, device=DEV)
    assert x.numel() > 2 ** 31
    x.fill_(1.0)
    hist = torch.full((B, 1), V - 1, dtype=torch.int32, device=DEV)
    one, none = (torch.full((B,), v, dtype=torch.int32, device=DEV) for v in (1, 0))
    K.apply_penalties(x, hist, none, one, presence=torch.full((B,), 0.5, device=DEV), out=x)
    assert (x[:, V - 1] == 0.5).all() and (x[:, :V - 1].amin(0) == 1).all() and (x[:, :V - 1].amax(0) == 1).all()


def test_graphs_streams_and_the_sampler():
    """Captured and replayed with eager work between, on another stream, and
    before the sampler, which then draws allowed tokens only."""
    rng = np.random.default_rng(8)
    B, V, L = 6, 32000, 100
    x = logits_of(rng, B, V)
    tokens, prompts, lens = (dev(t, np.int32) for t in (rng.integers(0, V, (B, L)), np.full(B, 3), np.full(B, L)))
    pen = [dev(np.full(B, v), np.float32) for v in (1.3, 0.5, 0.2)]
    allowed = rng.random((B, V)) < 0.001
    bits = dev(words(allowed), np.int32)
    run = lambda: K.apply_penalties(x, tokens, prompts, lens, *pen, allowed=bits)  # noqa: E731
    run()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = run()
    for turn in range(3):
        x.copy_(logits_of(rng, B, V))
        lens.fill_(L - 30 * turn)
        g.replay()
        assert torch.equal(o, run())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, o)
    u = torch.rand(B, device=DEV)
    for tok in (K.sample_filtered(o, torch.ones(B, device=DEV), u), K.sample_gumbel(o, torch.ones(B, device=DEV), 1, 0)):
        assert all(allowed[b, t] for b, t in enumerate(tok.tolist()))


def test_refusals():
    x = torch.zeros(2, 100, dtype=torch.bfloat16, device=DEV)
    i, f = torch.zeros(2, dtype=torch.int32, device=DEV), torch.ones(2, device=DEV)
    tokens = torch.zeros(2, 5, dtype=torch.int32, device=DEV)
    call = K.apply_penalties
    with pytest.raises(TypeError, match="logits"):
        call(x.half())
    with pytest.raises(ValueError, match="go together"):
        call(x, tokens, i)
    with pytest.raises(ValueError, match="need tokens"):
        call(x, presence=f)
    with pytest.raises(ValueError, match="bias_ids and bias"):
        call(x, bias_ids=tokens)
    with pytest.raises(TypeError, match="tokens"):
        call(x, tokens.long(), i, i)
    with pytest.raises(AssertionError, match="allowed"):
        call(x, allowed=torch.zeros(2, 3, dtype=torch.int32, device=DEV))
    with pytest.raises(AssertionError, match="repetition"):
        call(x, tokens, i, i, repetition=f[:1])
    with pytest.raises(ValueError, match="1024"):
        call(x, bias_ids=tokens.repeat(1, 300), bias=torch.zeros(2, 1500, device=DEV))
    with pytest.raises(ValueError, match="overlap"):
        call(x, out=x[:1].expand(2, 100))
    with pytest.raises(ValueError, match="GPU"):
        call(x, tokens.cpu(), i, i)
