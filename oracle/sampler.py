"""CPU restatement of the decode sampler (numpy).  TEST INFRASTRUCTURE.

sample_gumbel follows utils/sampler.py:35-53 of the reference:
    argmax( softmax(logits / T) / clamp(Exp(1) noise, 1e-10) )
with the noise supplied.  philox4x32_10 is the counter-based generator the
HIP sampler draws its noise from (Salmon, Moraes, Dror, Shaw, "Parallel
random numbers: as easy as 1, 2, 3", SC'11: 10 rounds of two 32x32->64-bit
multiplies by 0xD2511F53 / 0xCD9E8D57 with Weyl key increments 0x9E3779B9 /
0xBB67AE85), and exp_noise maps its words to Exp(1) variates exactly as the
kernel does: u = (w + 1) * 2^-32 in (0, 1], e = -log(u).

Pinning (tests/test_oracle_sampler.py): philox4x32_10 against the published
known-answer vectors of the Random123 distribution; sample_gumbel against a
brute-force scalar loop; the noise map against the Exp(1) moments.
"""
from __future__ import annotations

import numpy as np

M0, M1 = 0xD2511F53, 0xCD9E8D57
W0, W1 = 0x9E3779B9, 0xBB67AE85
MASK = 0xFFFFFFFF


def philox4x32_10(ctr, key):
    """ctr: 4 uint32 words (array-like [..., 4]); key: 2 uint32 words
    ([..., 2]).  Returns uint32 [..., 4]."""
    c = np.asarray(ctr, dtype=np.uint64).copy()
    k = np.asarray(key, dtype=np.uint64).copy()
    c0, c1, c2, c3 = c[..., 0], c[..., 1], c[..., 2], c[..., 3]
    k0, k1 = k[..., 0], k[..., 1]
    for r in range(10):
        if r:
            k0 = (k0 + W0) & MASK
            k1 = (k1 + W1) & MASK
        p0 = c0 * M0
        p1 = c2 * M1
        hi0, lo0 = p0 >> 32, p0 & MASK
        hi1, lo1 = p1 >> 32, p1 & MASK
        c0, c1, c2, c3 = (hi1 ^ c1 ^ k0) & MASK, lo1, (hi0 ^ c3 ^ k1) & MASK, lo0
    return np.stack([c0, c1, c2, c3], axis=-1).astype(np.uint32)


def noise_words(B, V, seed, offset):
    """The uint32 word of element (b, i): Philox with counter
    (i // 4 + offset_lo, offset_hi, b, 0x53414D50) and key (seed_lo, seed_hi),
    word i % 4 -- the layout of lfs_sample_gumbel."""
    i = np.arange(V, dtype=np.uint64)
    b = np.arange(B, dtype=np.uint64)
    lo = (i // 4 + (offset & MASK)) & MASK
    ctr = np.zeros((B, V, 4), np.uint64)
    ctr[..., 0] = lo[None, :]
    ctr[..., 1] = ((offset >> 32) & MASK) + ((i // 4 + (offset & MASK)) >> 32)[None, :]
    ctr[..., 2] = b[:, None]
    ctr[..., 3] = 0x53414D50
    key = np.array([seed & MASK, (seed >> 32) & MASK], np.uint64)
    out = philox4x32_10(ctr, np.broadcast_to(key, (B, V, 2)))
    return out[np.arange(B)[:, None], np.arange(V)[None, :], (i % 4).astype(np.int64)[None, :]]


def exp_noise(words):
    """u = (w + 1) * 2^-32 in (0, 1], e = -log(u) (float64)."""
    u = (np.asarray(words, np.float64) + 1.0) * 2.0 ** -32
    return -np.log(u)


def sample_gumbel(logits, temperatures, noise, dtype=np.float64):
    """utils/sampler.py:46-52: probs = softmax(logits / T); argmax(probs /
    clamp(noise, 1e-10)) per row (first index on ties)."""
    x = np.asarray(logits, dtype) / np.asarray(temperatures, dtype)[:, None]
    x = x - x.max(axis=1, keepdims=True)
    p = np.exp(x)
    p = p / p.sum(axis=1, keepdims=True)
    score = p / np.maximum(np.asarray(noise, dtype), 1e-10)
    return score.argmax(axis=1), score


def sample_filtered(logits, temperature, u, top_k=0, top_p=1.0, min_p=0.0):
    """One row in 64 bits: (token, log of its share of the kept weight).  The
    tokens are ordered by logit, largest first, equal ones by index; kept are
    the first top_k, of those the shortest prefix that reaches top_p of their
    weight, of those the ones with at least min_p of the largest weight; drawn
    is the first at which the kept weight summed so far exceeds u of it."""
    x = np.asarray(logits, np.float64)
    valid = np.flatnonzero(x > -np.inf)  # no NaN either
    if not len(valid):
        return 0, -np.inf
    order = valid[np.argsort(-x[valid], kind="stable")]
    if not temperature > 0:
        top_k, temperature = 1, 1.0
    s = x[order]
    with np.errstate(invalid="ignore"):
        e = np.where(s == s[0], 0.0, (s - s[0]) / np.float64(temperature))
    w = np.exp(np.where(np.isnan(e), -np.inf, e))
    n = min(top_k, len(w)) if top_k > 0 else len(w)
    c = np.cumsum(w[:n])
    if top_p < 1:
        n = max(1, int(np.count_nonzero(np.concatenate([[0.0], c[:-1]]) < top_p * c[-1])))
    if min_p > 0:
        n = max(1, min(n, int(np.count_nonzero(w >= min_p))))
    c = np.cumsum(w[:n])
    i = min(int(np.count_nonzero(c <= u * c[-1])), n - 1)
    return int(order[i]), e[i] - np.log(c[-1])


def apply_penalties(logits, history, prompt_len, repetition=None, presence=0.0, frequency=0.0, biases=(), allowed=None):
    """One row in 64 bits: repetition divides or multiplies the logits of the
    history's tokens, frequency and presence count those past the prompt,
    ``biases`` are (token, value) pairs, ``allowed`` truth values per token."""
    x = np.asarray(logits, np.float64).copy()
    V = len(x)
    history = [int(t) for t in history]
    if repetition is not None:
        for t in set(history):
            if 0 <= t < V:
                x[t] = x[t] / repetition if x[t] > 0 else x[t] * repetition
    for t in set(history[max(0, prompt_len):]):
        if 0 <= t < V:
            x[t] -= frequency * history[max(0, prompt_len):].count(t) + presence
    for t, value in biases:
        if 0 <= t < V:
            x[t] += value
    return x if allowed is None else np.where(allowed, x, -np.inf)
