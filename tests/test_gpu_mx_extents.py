"""GPU: microscaled weights of the most inputs and of the most outputs, over inputs whose results are known by arithmetic
(tests/mx_cut.py)."""
from __future__ import annotations

import numpy as np
import pytest

import mx_cut as X
from cogito_amd.capi import CGX_MX_FP4, CGX_MX_FP32, last_error
from gpu_util import device_tensor
from test_gpu_mx import Loss, Weight, _matmul, _within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 17, 70])
def test_most_inputs(gpu, M):
    """2^20 inputs: products split as far as they are, joined; losses of them; the gradient's second product over 4096 blocks."""
    K, N = 1 << 20, 19
    x, at, c, six = X.one_value_rows(M, K, N)
    w = Weight(gpu, X.pack4(c), np.full(c.shape[:2], 127, np.uint8), K, N, grad=1)
    x, at = x[0], at[0]
    h = np.zeros((M, K), np.float32)
    h[np.arange(M), at] = x
    z = x.astype(np.float64)[:, None] * X.weight_rows(c, at)
    _within(_matmul(gpu, w, h, K, N, CGX_MX_FP32) - z, X.ONE_VALUE * np.abs(z))
    t = np.where(np.arange(M) % 2, six[at], (six[at] + 1) % N).astype(np.int32)
    loss, lse, dh = Loss(gpu, w, h, t, CGX_MX_FP32, N).run()
    top, own = z.max(1), z[np.arange(M), t]
    _within(lse - top, (X.ONE_VALUE + 2.0 ** -24) * top)
    _within(loss - (top - own), X.ONE_VALUE * (top + np.abs(own)) + 2.0 ** -23 * (top - own))
    # all the mass is at the largest logit, but for e^-128 and what lse is off by: p within 2 (6 2^-23 + 2^-24) top of 1
    off = 2 * (X.ONE_VALUE + 2.0 ** -24) * top + 7 * 2.0 ** -23
    W = np.where(c > 7, -X.FP4[c & 7], X.FP4[c & 7]).reshape(N, -1)[:, :K].astype(np.float32)
    for m in range(M):
        want = W[six[at[m]]] - W[t[m]]
        assert np.all(np.abs(dh[m] - want) <= off[m] * (np.abs(W[six[at[m]]]) + np.abs(W[t[m]])) + 1e-37)


def test_most_outputs(gpu):
    """2^24 outputs of 33 inputs: offsets of codes, of parts and of several pieces of the vocabulary."""
    M, K, V = 3, 33, 1 << 24
    rng = np.random.default_rng(61)
    few = X.codes(rng, 1 << 12, K)
    few = np.where(few & 7 == 7, few - 1, few)
    c = np.tile(few, (V >> 12, 1, 1))
    best = np.array([V - 1, 5, V // 2 + 77])                 # the output of each row's largest logit
    at = np.array([32, 0, 31])
    c[best, at // 32, at % 32] = 7
    w = Weight(gpu, X.pack4(c), np.full((V, 2), 127, np.uint8), K, V, grad=1)
    h = np.zeros((M, K), np.float32)
    h[np.arange(M), at] = 96
    t = np.array([V - 1, V - 2, 12345], np.int32)
    col = X.weight_rows(c, at)
    y = _matmul(gpu, w, h, K, V, CGX_MX_FP4)
    np.testing.assert_array_equal(y, np.float32(96) * col.astype(np.float32))
    for act in (CGX_MX_FP4, CGX_MX_FP32):
        loss, lse, dh = Loss(gpu, w, h, t, act, V).run()
        # 96 and 576 are held exactly by any form; the second largest logit is 192 below: 2^24 e^-192 of it
        np.testing.assert_array_equal(lse, np.full(M, 576, np.float32))
        np.testing.assert_array_equal(loss, (576 - 96 * col[np.arange(M), t]).astype(np.float32))
        row = lambda v: np.where(c[v] > 7, -X.FP4[c[v] & 7], X.FP4[c[v] & 7]).reshape(-1)[:K]  # noqa: E731
        np.testing.assert_array_equal(dh, np.stack([row(best[m]) - row(t[m]) for m in range(M)]).astype(np.float32))


def test_a_tensor_of_the_most_inputs(gpu):
    """A matrix of 2^20 inputs quantised by the library: 2^15 blocks of 32."""
    K, N, M = 1 << 20, 3, 2
    rng = np.random.default_rng(62)
    W = rng.choice(np.array([-4, -1, 0, 0.5, 2, 4], np.float32), (K, N))
    W[::32] = 4                                              # each block's scale is 1: its values are held exactly
    t = device_tensor(gpu, W)
    ptr = gpu.cgx_mx_weight_from_tensor(t, 0)
    assert ptr, last_error(gpu)
    w = Weight.__new__(Weight)
    w.lib, w.ptr = gpu, ptr
    h = np.zeros((M, K), np.float32)
    h[0, K - 1], h[1, K // 2 + 5] = 3, -7
    y = _matmul(gpu, w, h, K, N, CGX_MX_FP32)
    np.testing.assert_array_equal(y, np.stack([3 * W[K - 1], -7 * W[K // 2 + 5]]))
    gpu.cg_tensor_free(t)
