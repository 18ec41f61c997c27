"""GPU: every form of the kernels of microscaled products, the losses and the gradient (tests/mx_forms.py), over inputs
whose results show each of the terms that fp32 rows and probabilities are cut into (tests/mx_cut.py), and over dense ones.
Bounds of the dense ones: those of test_gpu_mx.py."""
from __future__ import annotations

import numpy as np
import pytest

import mx_cut as X
import mx_forms as F
import mx_ref as R
from cogito_amd.capi import CGX_MX_FP4, CGX_MX_FP32
from test_gpu_mx import ACTS, Loss, Weight, _check, _matmul, _ok, _rows, _targets, _tol, _within

pytestmark = pytest.mark.gpu
ALL = F.SEGMENTS + F.BLOCKS + [s for pair in F.BORDERS for s in pair] + [(M, 200, N) for N, _ in F.TILES for M in F.FEW]


def _handle(gpu, c, N, K, grad=0):
    return Weight(gpu, X.pack4(c), np.full(c.shape[:2], 127, np.uint8), K, N, grad=grad)


# ------------------------------------------------------- the small terms

@pytest.mark.parametrize("M,K,N", ALL)
def test_one_value_of_a_row(gpu, M, K, N):
    """Products and losses of rows of one value each, at inputs spread over the whole contraction."""
    x, at, c, six = X.one_value_rows(M, K, N, reps=-(-24 // M))
    w = _handle(gpu, c, N, K)
    rng = np.random.default_rng(N)
    for x, at in zip(x, at):
        h = np.zeros((M, K), np.float32)
        h[np.arange(M), at] = x
        z = x.astype(np.float64)[:, None] * X.weight_rows(c, at)
        y = _matmul(gpu, w, h, K, N, CGX_MX_FP32)
        _within(y - z, X.ONE_VALUE * np.abs(z))
        # the second largest logit is at least 2 * 64 below: e^-128 of it
        t = rng.integers(0, N, M).astype(np.int32)
        loss, lse, _ = Loss(gpu, w, h, t, CGX_MX_FP32, N, grad=False).run()
        top, own = z[np.arange(M), six[at]], z[np.arange(M), t]
        _within(lse - top, (X.ONE_VALUE + 2.0 ** -24) * top)
        _within(loss - (top - own), X.ONE_VALUE * (top + np.abs(own)) + 2.0 ** -23 * (top - own))


# the gradient: probabilities in the epilogue of row blocks of 16, 32, 64 and 128 rows and of split products' sums; the second
# product in row blocks of 16, 32 and 64, split and whole, double-buffered and not; several pieces of the vocabulary; slabs
GRADIENTS = [(1, 64, 64), (5, 700, 700), (16, 2100, 2100), (20, 2100, 2100), (33, 300, 5000), (40, 96, 3000), (61, 768, 50257), (100, 2500, 2600),
             (300, 512, 27000), (1024, 300, 16400), (600, 40, 60000), (2048 + 70, 33, 700), (7, 9000, 9000)]


@pytest.mark.parametrize("act", [CGX_MX_FP4, CGX_MX_FP32])
@pytest.mark.parametrize("M,K,V", GRADIENTS)
def test_one_probability_of_an_input(gpu, M, K, V, act):
    h, of, c, lse, t, dh, tol, _ = X.one_output_inputs(M, K, V, lambda a: R.taken(a, act))
    g = np.random.default_rng(V).normal(size=M).astype(np.float32)
    call = Loss(gpu, _handle(gpu, c, V, K, grad=1), h, t, act, V, g)
    call.lse.upload(np.concatenate([lse, np.full(4, 7, np.float32)]))
    _ok(gpu, call.backward())
    _within(call.read()[2] - g[:, None] * dh, np.abs(g)[:, None] * tol)


# ------------------------------------------------------------ dense rows

def _dense(rng, N, K, size):
    """Codes, bytes and W of random codes over scales two powers of two apart."""
    c = X.codes(rng, N, K)
    b = (127 + int(np.floor(np.log2(size))) - rng.integers(0, 3, c.shape[:2])).astype(np.uint8)
    return c, b, R.values(c, b, 4, K).T


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("N", [n for n, _ in F.TILES])
def test_tiles_of_a_block(gpu, N, act):
    """Few rows over every count of tiles a block takes: the product, and the loss over it."""
    rng = np.random.default_rng(N + act)
    K = 200
    c, b, W = _dense(rng, N, K, 1 / 16)
    w = Weight(gpu, X.pack4(c), b, K, N)
    for M in F.FEW:
        h, t = _rows(rng, M, K), _targets(rng, M, N)
        x = R.taken(h, act)
        _within(_matmul(gpu, w, h, K, N, act, ldy=N + 1) - x @ W, _tol(np.abs(x), R.cut_error(h, act), W, K, act))
        _check(Loss(gpu, w, h, t, act, N, ldh=K + 3, grad=False).run(), h, W, t, act, grad=False)


@pytest.mark.parametrize("M,K,N", F.SEGMENTS[:4])
def test_segments_of_few_rows(gpu, M, K, N):
    rng = np.random.default_rng(M + K + N)
    c, b, W = _dense(rng, N, K, 1.5 / np.sqrt(K))
    w = Weight(gpu, X.pack4(c), b, K, N)
    h, t = _rows(rng, M, K), _targets(rng, M, N)
    _within(_matmul(gpu, w, h, K, N, CGX_MX_FP32) - h.astype(np.float64) @ W, _tol(np.abs(h), R.cut_error(h, 32), W, K, CGX_MX_FP32))
    _check(Loss(gpu, w, h, t, CGX_MX_FP32, N, grad=False).run(), h, W, t, CGX_MX_FP32, grad=False)


@pytest.mark.parametrize("factor", [1e3, 1e5])
@pytest.mark.parametrize("M", [3, 40])
def test_rows_with_outlier_channels(gpu, M, factor):
    """fp32 rows are held to 2^-23 of the largest value of a block of 32, not each to its own: a channel that is `factor` times
    the others costs its 31 neighbours as much of their precision, whether or not its own weight counts.  Outputs that the
    outliers do not enter (weights of 0) are off by that much and no more."""
    rng = np.random.default_rng(51)
    K, N = 4096, 200
    c, b, _ = _dense(rng, N, K, 0.02)
    c[:, :, 9] = 0
    W = R.values(c, b, 4, K).T
    x = rng.normal(size=(M, K)).astype(np.float32)
    x[:, 9::32] *= np.float32(factor)
    y = _matmul(gpu, Weight(gpu, X.pack4(c), b, K, N), x, K, N, CGX_MX_FP32)
    exp, rest = x.astype(np.float64) @ W, np.abs(x.astype(np.float64))
    rest[:, 9::32] = 0
    _within(y - exp, _tol(rest, R.cut_error(x, 32), W, K, CGX_MX_FP32))
