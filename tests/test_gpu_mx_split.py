"""GPU: losses and gradients over vocabularies of few blocks, whose contraction is split and whose logits' parts are added up
by a launch of their own.  Bounds: those of test_gpu_mx.py."""
from __future__ import annotations

import numpy as np
import pytest

import mx_ref as R
from cogito_amd.capi import CGX_MX_FP4, CGX_MX_FP6, CGX_MX_FP32, last_error
from test_gpu_mx import ACTS, Loss, Weight, _check, _ok, _rows, _targets, _up

pytestmark = pytest.mark.gpu


# K from where a contraction is split at all (16 chunks of 128) to many splits; V of 1, odd, of several segments of 1024;
# rows of less than a tile, of a tile and one, of many row blocks
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows,K,V", [(1, 4096, 33), (16, 4096, 300), (17, 2048, 1), (20, 4097, 500), (30, 4000, 4001), (84, 2500, 4620), (130, 4100, 1001),
                                      (300, 4096, 129), (5, 20000, 260)])
def test_losses_of_split_contractions(gpu, rows, K, V, act):
    rng = np.random.default_rng(rows + K + V)
    codes, byte, W = R.weight(rng, V, K, 1.5 / np.sqrt(K))
    h, t = _rows(rng, rows, K), _targets(rng, rows, V)
    g = rng.normal(size=rows).astype(np.float32)
    c = Loss(gpu, Weight(gpu, codes, byte, K, V, grad=1), h, t, act, V, g, ldh=K + 3, ldd=K + 1)
    out = c.run()
    _check(out, h, W, t, act, g)
    ignored = (t < 0) | (t >= V)
    assert np.all(out[0][ignored] == 0) and np.all(out[2][ignored] == 0)
    for a, b in zip(c.run(), out):
        np.testing.assert_array_equal(a, b)


def test_split_losses_of_extreme_rows(gpu):
    rng = np.random.default_rng(17)
    K, V, n = 4096, 400, 24
    codes, byte, W = R.weight(rng, V, K, 1.0 / 8)
    h = _rows(rng, n, K)
    t = rng.integers(0, V, n).astype(np.int32)
    h[1] = 0                                           # uniform
    h[2] *= 300                                        # one token has all the mass
    h[3, 5], h[4, 4095] = np.nan, np.inf
    h[5] *= np.float32(1e-30)
    t[7], h[7, 0] = -1, np.nan                         # an ignored row
    t[2] = int((h[2].astype(np.float64) @ W).argmax())
    loss, lse, dh = Loss(gpu, Weight(gpu, codes, byte, K, V, grad=1), h, t, CGX_MX_FP32, V).run()
    assert np.all(np.isnan(lse[[3, 4, 7]])) and np.all(np.isnan(loss[[3, 4]])) and np.all(np.isnan(dh[[3, 4]]))
    assert loss[7] == 0 and np.all(dh[7] == 0)
    ok = [i for i in range(n) if i not in (3, 4, 7)]
    _check((loss[ok], lse[ok], dh[ok]), h[ok], W, t[ok], CGX_MX_FP32)


def test_a_weight_block_without_a_value(gpu):
    """A weight's block of byte 255 makes every row's loss and gradient NaN, whichever split holds it."""
    rng = np.random.default_rng(18)
    K, V, n = 4096, 300, 20
    codes, byte, _ = R.weight(rng, V, K, 0.02)
    byte = byte.copy()
    byte[123, 77] = 255
    h = _rows(rng, n, K)
    t = rng.integers(0, V, n).astype(np.int32)
    t[3] = -1
    loss, lse, dh = Loss(gpu, Weight(gpu, codes, byte, K, V, grad=1), h, t, CGX_MX_FP32, V).run()
    live = np.arange(n) != 3
    assert np.all(np.isnan(lse)) and np.all(np.isnan(loss[live])) and loss[3] == 0
    assert np.all(np.isnan(dh[live])) and np.all(dh[3] == 0)


def test_split_losses_captured_over_one_workspace(gpu):
    rng = np.random.default_rng(19)
    K, V = 4096, 700
    codes, byte, W = R.weight(rng, V, K, 0.02)
    w = Weight(gpu, codes, byte, K, V, grad=1)
    sets = [Loss(gpu, w, _rows(rng, n, K), _targets(rng, n, V), act, V)
            for n, act in ((3, CGX_MX_FP32), (40, CGX_MX_FP4), (70, CGX_MX_FP32), (20, CGX_MX_FP6))]
    need = max(c.need for c in sets)
    ws = _up(gpu, np.full(need + 256, 0xC3), np.uint8)
    first = []
    for c in sets:
        c.ws, c.need = ws, need
        first.append([x.copy() for x in c.run()])
    graphs = []
    for c in sets:
        assert gpu.cgx_graph_begin() == 0
        rc = c.forward() or c.backward()
        graphs.append(gpu.cgx_graph_end())
        assert rc == 0 and graphs[-1], last_error(gpu)
    for _ in range(3):
        for c, g, want in zip(sets, graphs, first):
            for x in (c.loss, c.lse, c.dh):
                _ok(gpu, gpu.cgx_memset(x.ptr, 0, x.nbytes - 16))
            _ok(gpu, gpu.cgx_graph_launch(g))
            _ok(gpu, gpu.cgx_synchronize())
            for a, b in zip(c.read(), want):
                np.testing.assert_array_equal(a, b)
    for g in graphs:
        gpu.cgx_graph_free(g)
