"""GPU: microscaled products and losses as a program calls them: captured and replayed, in a row over one
workspace, through pieces and slabs, over long and far arrays, and with the operators beside them.  Bounds: those
of test_gpu_mx.py."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import mx_ref as R
from cogito_amd.capi import CGX_MX_FP4, CGX_MX_FP6, CGX_MX_FP32, DeviceArray, last_error
from gpu_util import device_tensor
from test_gpu_mx import Loss, Weight, _check, _matmul, _ok, _rows, _targets, _tol, _up, _within

pytestmark = pytest.mark.gpu


# rows that go over the kernel of few rows in one segment and in several, and the other's row blocks, split and whole
@pytest.mark.parametrize("act", [CGX_MX_FP4, CGX_MX_FP32])
@pytest.mark.parametrize("M,K,N", [(1, 11008, 300), (7, 11008, 130), (8, 11008, 130), (16, 5120, 100), (16, 5121, 100), (11, 4096, 4200), (16, 2176, 33000),
                                   (2, 256, 70000), (33, 4000, 600), (100, 2100, 5000), (513, 140, 30000), (640, 130, 33000)])
def test_products_of_other_shapes(gpu, M, K, N, act):
    rng = np.random.default_rng(M + K + N)
    codes, byte, W = R.weight(rng, N, K, 0.1, 2)
    x = _rows(rng, M, K)
    w = Weight(gpu, codes, byte, K, N)
    y = _matmul(gpu, w, x, K, N, act)
    xt = R.taken(x, act)
    _within(y - xt @ W, _tol(np.abs(xt), R.cut_error(x, act), W, K, act))
    np.testing.assert_array_equal(_matmul(gpu, w, x, K, N, act), y)


@pytest.mark.parametrize("rows,K,V", [(3, 8000, 300), (12, 8000, 300), (600, 40, 60000), (2048 + 70, 33, 700), (129, 64, 33000), (1025, 128, 4100), (16, 64, 40000)])
def test_losses_of_other_shapes(gpu, rows, K, V):
    """Long rows, more rows than a slab holds, vocabularies in more than one piece."""
    rng = np.random.default_rng(rows + V)
    codes, byte, W = R.weight(rng, V, K, 1.5 / np.sqrt(K))
    h, t = _rows(rng, rows, K), _targets(rng, rows, V)
    g = rng.normal(size=rows).astype(np.float32)
    c = Loss(gpu, Weight(gpu, codes, byte, K, V, grad=1), h, t, CGX_MX_FP32, V, g)
    out = c.run()
    _check(out, h, W, t, CGX_MX_FP32, g)
    for a, b in zip(c.run(), out):
        np.testing.assert_array_equal(a, b)


def test_graphs_share_a_workspace(gpu):
    """Captured products, losses and gradients over one workspace, replayed in turn behind eager calls: the same bits every time."""
    rng = np.random.default_rng(31)
    K, V = 700, 3000
    codes, byte, W = R.weight(rng, V, K, 0.05)
    w = Weight(gpu, codes, byte, K, V, grad=1)
    sets = []
    for n, act in ((3, CGX_MX_FP32), (40, CGX_MX_FP4), (70, CGX_MX_FP32), (200, CGX_MX_FP6)):
        h, t = _rows(rng, n, K), _targets(rng, n, V)
        c = Loss(gpu, w, h, t, act, V)
        c.y = DeviceArray(gpu, n * V * 4)
        sets.append(c)
    need = max([c.need for c in sets] + [gpu.cgx_matmul_mx_ws(w.ptr, c.n, c.act) for c in sets])
    ws = _up(gpu, np.full(need + 256, 0xC3), np.uint8)
    for c in sets:
        c.ws, c.need = ws, need

    def call(c):
        return gpu.cgx_matmul_mx_dev(c.h.ptr, K, c.n, w.ptr, c.act, c.y.ptr, V, ws.ptr, need) or c.forward() or c.backward()

    def bits(c):
        return [x.copy() for x in c.read()] + [c.y.numpy(np.uint32, (c.n * V,))]
    first = []
    for c in sets:
        _ok(gpu, call(c))
        first.append(bits(c))
    graphs = []
    for c in sets:
        assert gpu.cgx_graph_begin() == 0
        rc = call(c)
        graphs.append(gpu.cgx_graph_end())
        assert rc == 0 and graphs[-1], last_error(gpu)
    for turn in range(3):
        for i, c in enumerate(sets):
            other = sets[(i + turn + 1) % len(sets)]
            for d in (c.loss, c.lse, c.dh, c.y):
                d.upload(np.full(min(d.nbytes // 4, c.n), 7, np.float32))
            c.dh.upload(np.full(c.n * c.ldd + 4, 7, np.float32))
            c.loss.upload(np.full(c.n + 4, 7, np.float32))
            c.lse.upload(np.full(c.n + 4, 7, np.float32))
            assert gpu.cgx_graph_launch(graphs[i]) == 0
            _ok(gpu, call(other))
            for k, x in ((i, c), (sets.index(other), other)):
                for a, b in zip(bits(x), first[k]):
                    np.testing.assert_array_equal(a.view(np.uint32) if a.dtype == np.float32 else a,
                                                  b.view(np.uint32) if b.dtype == np.float32 else b)
    for g in graphs:
        assert gpu.cgx_graph_free(g) == 0


def test_a_smaller_call_in_the_workspace_of_a_larger(gpu):
    rng = np.random.default_rng(32)
    K, V, most = 400, 2000, 300
    codes, byte, W = R.weight(rng, V, K, 0.07)
    w = Weight(gpu, codes, byte, K, V, grad=1)
    h, t = _rows(rng, most, K), _targets(rng, most, V)
    n = gpu.cgx_token_loss_mx_ws(w.ptr, most, CGX_MX_FP32, 1)
    ws = _up(gpu, np.full(n + 256, 0xC3), np.uint8)
    for rows in (300, 299, 129, 64, 33, 17, 16, 5, 1):
        c = Loss(gpu, w, h[:rows], t[:rows], CGX_MX_FP32, V)
        c.ws, c.need = ws, n
        _check(c.run(), h[:rows], W, t[:rows], CGX_MX_FP32)


def test_outputs_beyond_four_gigabytes(gpu):
    """Rows of y so far apart that the last lie beyond 2^32 bytes."""
    rng = np.random.default_rng(33)
    M, K, N, ld = 70, 96, 200, 20_000_000
    codes, byte, W = R.weight(rng, N, K)
    x = _rows(rng, M, K)
    w = Weight(gpu, codes, byte, K, N)
    d, y = _up(gpu, x, np.float32), DeviceArray(gpu, ((M - 1) * ld + N) * 4)
    n = gpu.cgx_matmul_mx_ws(w.ptr, M, CGX_MX_FP32)
    ws = DeviceArray(gpu, n)
    _ok(gpu, gpu.cgx_matmul_mx_dev(d.ptr, K, M, w.ptr, CGX_MX_FP32, y.ptr, ld, ws.ptr, n))
    got = np.empty((M, N), np.float32)
    for m in range(M):
        assert gpu.cgx_memcpy_d2h(got[m].ctypes.data, y.ptr + m * ld * 4, N * 4) == 0
    _within(got - x.astype(np.float64) @ W, _tol(np.abs(x), R.cut_error(x, 32), W, K, CGX_MX_FP32))


def test_weights_beyond_four_gigabytes(gpu):
    """A weight of 2^33 values: every code 1.0 but those of the last outputs, which only offsets in 64 bits reach."""
    K, N = 4096, 1 << 21
    codes, scales = DeviceArray(gpu, N * K // 2), DeviceArray(gpu, N * K // 32)
    assert gpu.cgx_memset(codes.ptr, 0x22, codes.nbytes) == 0 and gpu.cgx_memset(scales.ptr, 127, scales.nbytes) == 0
    last = np.full(K // 2, 0x55, np.uint8)                        # 3.0
    assert gpu.cgx_memcpy_h2d(codes.ptr + codes.nbytes - K // 2, last.ctypes.data, K // 2) == 0
    w = gpu.cgx_mx_weight_new(codes.ptr, scales.ptr, K, N, 0)
    assert w, last_error(gpu)
    codes.free()
    scales.free()
    x = np.ones((2, K), np.float32)
    x[1] = 0.5
    d, y = _up(gpu, x, np.float32), DeviceArray(gpu, 2 * N * 4)
    n = gpu.cgx_matmul_mx_ws(w, 2, CGX_MX_FP32)
    ws = DeviceArray(gpu, n)
    _ok(gpu, gpu.cgx_matmul_mx_dev(d.ptr, K, 2, w, CGX_MX_FP32, y.ptr, N, ws.ptr, n))
    got = y.numpy(np.float32, (2, N))
    assert np.all(got[0, :-1] == K) and np.all(got[1, :-1] == K / 2) and got[0, -1] == 3 * K and got[1, -1] == 1.5 * K
    gpu.cgx_mx_weight_free(w)


def test_a_scored_prompt(gpu):
    """Rows through two weights made from matrices, then the prompt's losses: those of the log probabilities of the logits that
    the product gives."""
    rng = np.random.default_rng(34)
    n, K, D, V = 37, 320, 256, 5000
    a, b = rng.normal(size=(K, D)).astype(np.float32) / 18, rng.normal(size=(D, V)).astype(np.float32) / 16
    ta, tb = device_tensor(gpu, a), device_tensor(gpu, b)
    wa, wb = gpu.cgx_mx_weight_from_tensor(ta, 0), gpu.cgx_mx_weight_from_tensor(tb, 1)
    assert wa and wb, last_error(gpu)
    x, t = _rows(rng, n, K), rng.integers(0, V, n).astype(np.int32)
    need = max(gpu.cgx_matmul_mx_ws(wa, n, CGX_MX_FP6), gpu.cgx_matmul_mx_ws(wb, n, CGX_MX_FP32), gpu.cgx_token_loss_mx_ws(wb, n, CGX_MX_FP32, 1),
               gpu.cgx_token_logprobs_ws(n, V, 0))
    ws, dx, dt = DeviceArray(gpu, need), _up(gpu, x, np.float32), _up(gpu, t, np.int32)
    h, z, lp, loss, lse, dh = (DeviceArray(gpu, 4 * k) for k in (n * D, n * V, n, n, n, n * D))
    _ok(gpu, gpu.cgx_matmul_mx_dev(dx.ptr, K, n, wa, CGX_MX_FP6, h.ptr, D, ws.ptr, need) or
        gpu.cgx_matmul_mx_dev(h.ptr, D, n, wb, CGX_MX_FP32, z.ptr, V, ws.ptr, need) or
        gpu.cgx_token_logprobs_dev(z.ptr, V, n, V, dt.ptr, 0, lp.ptr, None, None, None, None, ws.ptr, need) or
        gpu.cgx_token_loss_mx_dev(h.ptr, D, n, wb, CGX_MX_FP32, dt.ptr, loss.ptr, lse.ptr, ws.ptr, need) or
        gpu.cgx_token_loss_mx_grad_dev(h.ptr, D, n, wb, CGX_MX_FP32, dt.ptr, lse.ptr, None, dh.ptr, D, ws.ptr, need))
    WA, WB = (R.values(*R.quantise(m.T, 4), 4, m.shape[0]).T for m in (a, b))
    hid = h.numpy(np.float32, (n, D))
    xt = R.taken(x, CGX_MX_FP6)
    _within(hid - xt @ WA, _tol(np.abs(xt), np.zeros(x.shape), WA, K, CGX_MX_FP6))
    out = (loss.numpy(np.float32, (n,)), lse.numpy(np.float32, (n,)), dh.numpy(np.float32, (n, D)))
    _check(out, hid, WB, t, CGX_MX_FP32)
    # both from logits within T; the log probability's own bound is 6e-6 + 2^-23 of it
    T = _tol(np.abs(hid), R.cut_error(hid, 32), WB, D, CGX_MX_FP32).max(1)
    _within(lp.numpy(np.float32, (n,)) + out[0], 4 * T + 6e-6 + 2.0 ** -17 + 2.0 ** -21 * np.abs(out[0]))
    for p in (wa, wb):
        gpu.cgx_mx_weight_free(p)
    gpu.cg_tensor_free(ta)
    gpu.cg_tensor_free(tb)


def test_quantised_rows_are_what_the_product_takes(gpu):
    """The product of rows that were quantised and read back is that of the rows themselves, bit for bit."""
    rng = np.random.default_rng(35)
    n, K, N = 21, 210, 90
    codes, byte, _ = R.weight(rng, N, K)
    w = Weight(gpu, codes, byte, K, N)
    x = _rows(rng, n, K)
    d, back = _up(gpu, x, np.float32), DeviceArray(gpu, n * K * 4)
    for fmt in (CGX_MX_FP4, CGX_MX_FP6):
        c, s = DeviceArray(gpu, n * 7 * 24), DeviceArray(gpu, n * 7)
        _ok(gpu, gpu.cgx_mx_quantize_dev(d.ptr, K, n, K, fmt, c.ptr, s.ptr) or
            gpu.cgx_mx_dequantize_dev(c.ptr, s.ptr, n, K, fmt, back.ptr, K))
        np.testing.assert_array_equal(_matmul(gpu, w, back.numpy(np.float32, (n, K)), K, N, fmt), _matmul(gpu, w, x, K, N, fmt))


@pytest.mark.parametrize("rows,K", [(3, 32), (20, 32), (20, 4096)])
def test_logits_at_the_ends_of_the_range(gpu, rows, K):
    """Logits up to 3 2^126, exact: no difference of theirs leaves the range unnoticed."""
    V = 300
    w = np.zeros((V, K), np.float32)
    w[:, 0] = 0.5
    w[7, 0], w[9, 1], w[:, 2], w[11, 3] = 2, 3, -3, -3
    c, b = R.quantise(w, 4)
    h = np.zeros((rows, K), np.float32)
    big = np.float32(2.0 ** 126)
    h[0, 0] = h[1, 1] = h[2, 2] = big
    if rows > 3:
        h[3, 3] = big
        h[5, 0], h[6, 0] = 2.0 ** 40, 2.0 ** 24
    t = np.full(rows, 7, np.int32)
    loss, lse, dh = Loss(gpu, Weight(gpu, R.pack(c, 4), b, K, V, grad=1), h, t, CGX_MX_FP32, V).run()
    assert lse[0] == 2 * big and loss[0] == 0 and np.all(dh[0] == 0)
    assert lse[1] == 3 * big and loss[1] == 3 * big and dh[1, 1] == 3 and dh[1, 0] == 0.5 - 2
    assert lse[2] == -3 * big
    if rows > 3:
        # one token of no mass, 299 alike: off by the fp32 sums of 300 terms and lse's rounding
        assert abs(lse[3] - np.log(299.0)) < 2.0 ** -15 and abs(loss[3] - np.log(299.0)) < 2.0 ** -15
        assert abs(lse[4] - np.log(300.0)) < 2.0 ** -15
        assert lse[5] == 2.0 ** 41 and lse[6] == 2.0 ** 25 and not loss[5:7].any() and not dh[5:7].any()


@pytest.mark.parametrize("act", [CGX_MX_FP4, CGX_MX_FP6, CGX_MX_FP32])
@pytest.mark.parametrize("M,K,N,ld", [(12, 2229, 600, 2230), (1, 3611, 100, 3611), (7, 10001, 90, 10003), (16, 31, 70, 40), (3, 97, 4100, 98), (16, 5089, 33, 5100)])
def test_few_rows_that_end_inside_a_block(gpu, M, K, N, ld, act):
    """NaN behind every row; rows at any alignment; over one segment of the contraction and several."""
    rng = np.random.default_rng(M * K + N)
    codes, byte, W = R.weight(rng, N, K, 0.1, 2)
    x = _rows(rng, M, K)
    y = _matmul(gpu, Weight(gpu, codes, byte, K, N), x, K, N, act, ldx=ld, ldy=N + 1, offx=1, offy=3)
    xt = R.taken(x, act)
    _within(y - xt @ W, _tol(np.abs(xt), R.cut_error(x, act), W, K, act))


def test_blocks_captured(gpu):
    """Quantisation and read-back replayed over other values at the same addresses."""
    rng = np.random.default_rng(36)
    n, K = 37, 1000
    d, c, s, back = (DeviceArray(gpu, b) for b in (n * K * 4, n * 32 * 24, n * 32, n * K * 4))
    for fmt in (CGX_MX_FP4, CGX_MX_FP6):
        d.upload(_rows(rng, n, K))
        assert gpu.cgx_graph_begin() == 0
        rc = gpu.cgx_mx_quantize_dev(d.ptr, K, n, K, fmt, c.ptr, s.ptr) or gpu.cgx_mx_dequantize_dev(c.ptr, s.ptr, n, K, fmt, back.ptr, K)
        graph = gpu.cgx_graph_end()
        assert rc == 0 and graph, last_error(gpu)
        for _ in range(3):
            x = _rows(rng, n, K)
            d.upload(x)
            assert gpu.cgx_graph_launch(graph) == 0
            _ok(gpu, 0)
            got = back.numpy(np.float32, (n, K)).copy()
            np.testing.assert_array_equal(got, R.taken(x, fmt).astype(np.float32))
            _ok(gpu, gpu.cgx_mx_quantize_dev(d.ptr, K, n, K, fmt, c.ptr, s.ptr) or gpu.cgx_mx_dequantize_dev(c.ptr, s.ptr, n, K, fmt, back.ptr, K))
            np.testing.assert_array_equal(back.numpy(np.float32, (n, K)), got)
        assert gpu.cgx_graph_free(graph) == 0
