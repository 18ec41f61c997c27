"""Inputs whose results depend on the smallest of the terms that fp32 rows and probabilities are cut into, and the cut itself
in 64 bits with any number of terms (numpy; no code of the library).

Dense rows cannot show a missing term: sums over thousands of inputs are allowed more than it adds.  Here one value of a row,
or one probability, decides an output alone, so that nothing but its own terms and their sum is rounded."""
from __future__ import annotations

import numpy as np

FP4 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
SHIFTS = (0, 3, 8, 13, 18)                                   # powers of two of the terms below the block's


def cut(x, terms=5):
    """x [..., n] as held by that many 6-bit terms of each block of 32."""
    n = x.shape[-1]
    v = np.pad(np.asarray(x, np.float64), [(0, 0)] * (x.ndim - 1) + [(0, -n % 32)]).reshape(*x.shape[:-1], -1, 32)
    top = np.abs(v).max(-1, keepdims=True)
    e = np.maximum(np.frexp(np.where(top == 0, 2.0 ** -126, top))[1] - 1 - 2, 19 - 127)
    held = np.zeros_like(v)
    for s in SHIFTS[:terms]:
        scale = np.exp2((e - s).astype(np.float64))
        a = np.abs(v - held) / scale
        step = np.where(a < 2, 0.125, np.where(a < 4, 0.25, 0.5))
        held += np.copysign(np.minimum(np.rint(a / step) * step, 7.5), v - held) * scale
    return held.reshape(*x.shape[:-1], -1)[..., :n]


def pack4(c):
    """Bytes [N][blocks * 16] of 4-bit codes [N][blocks][32], the first in the lowest bits."""
    return (c[..., 0::2] | c[..., 1::2] << 4).reshape(len(c), -1)


def codes(rng, N, K, top=16):
    """Random codes below top in either sign [N][blocks][32], 0 past K."""
    c = rng.integers(0, top, (N, -(-K // 32), 32), dtype=np.uint8)
    if K % 32:
        c[:, -1, K % 32:] = 0
    return c


# ---------------------------------------------------- one value a row

def one_value_rows(M, K, N, reps=1):
    """Rows with one value of 24 bits between 64 and 100 at input at[r], spread over the whole of K, [reps][M]: of 200 drawn for
    each, the one that four terms hold worst.  The weight is 6 at one output of each input and at most 4 in magnitude elsewhere,
    over powers of two of 1: a row's largest logit is 128 above the rest, so that its log sum of exponentials is that logit.
    Returns values, at, codes and the outputs of 6."""
    rng = np.random.default_rng(M * 31 + K * 7 + N)
    x = rng.uniform(64, 100, (200, reps * M, 1)).astype(np.float32)
    x = np.take_along_axis(x, np.abs(cut(x, 4) / x - 1).argmax(0)[None], 0).reshape(reps, M)
    at = (np.linspace(0, K - 1, reps * M).astype(int) if reps * M > 1 else np.array([K - 1])).reshape(reps, M)
    at[-1, -1] = K - 1
    c = codes(rng, N, K)
    c = np.where(c & 7 == 7, c - 1, c)
    six = rng.integers(0, N, K)
    c[six, np.arange(K) // 32, np.arange(K) % 32] = 7
    return x, at, c, six


def weight_rows(c, at):
    """Weights of the inputs `at`, [len(at)][N]."""
    q = c[:, at // 32, at % 32].T
    return FP4[q & 7] * np.where(q > 7, -1.0, 1.0)


# the sum of a value's five terms over the weight: five instructions within 2^-23 of it each, and what the terms leave, 2^-23
ONE_VALUE = 6 * 2.0 ** -23


# ----------------------------------------------- one probability an input

def one_output_inputs(M, K, V, taken):
    """A weight with 1.0 at one output of each input (output of[k]) and 0 elsewhere, hidden rows of multiples of 1 / 256 up
    to 1.5, a log sum of exponentials of 2 that is given to the gradient, and targets, so that dh[m][k] = p - [of[k] is the
    target], p = exp(z - 2), z the row's own value as `taken` gives it.  Returns h, of, codes, lse, targets, dh and the
    bound of its error."""
    rng = np.random.default_rng(M + K * 5 + V * 3)
    h = (rng.integers(-384, 385, (M, K)) / 256).astype(np.float32)
    of = np.sort(rng.permutation(V)[:K])
    c = np.zeros((V, -(-K // 32), 32), np.uint8)
    c[of, np.arange(K) // 32, np.arange(K) % 32] = 2
    lse = np.full(M, 2.0, np.float32)
    t = rng.integers(0, V, M).astype(np.int32)
    t[::3] = of[rng.integers(0, K, len(t[::3]))]
    z = np.zeros((M, V))
    z[:, of] = taken(h)
    d = z - 2.0
    p = np.exp(d)
    q = p.copy()
    q[np.arange(M), t] -= 1
    # p: the logit's five terms, 2^-23 of it each; the exponent's product and its constant, 2^-24 and 2^-26 of it; 2^x to 2^-23,
    # expm1 to 2^-22.  Its terms hold 2^-23 of the largest of 32 outputs.  Five instructions sum them, 6 2^-23 of the value.
    # A last rounding, 2^-24.
    block = np.pad(np.abs(q), ((0, 0), (0, -V % 32))).reshape(M, -1, 32).max(2)
    off = p * (5 * 2.0 ** -23 * np.abs(z) + (2.0 ** -24 + 2.0 ** -26) * np.abs(d) + 2.0 ** -23)
    off += np.repeat(block, 32, 1)[:, :V] * 2.0 ** -23 + np.abs(q) * (6 * 2.0 ** -23 + 2.0 ** -24)
    off[np.arange(M), t] += np.abs(q[np.arange(M), t]) * 2.0 ** -22
    return h, of, c, lse, t, q[:, of], off[:, of], q
