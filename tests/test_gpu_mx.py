"""GPU: microscaled blocks, the product of rows with a 4-bit weight, and the loss over a vocabulary of it,
against 64 bits.

Tolerances.  A product's terms are exact in the matrix cores' products; what is rounded: the rows as they
are held (mx_ref.cut_error, times |W|), and fp32 sums.  One instruction adds 128 terms to the sum within
2^-23 of the sum of magnitudes (measured 2^-23.4 at most); a row of K inputs takes n = ceil(K / 128) of them for each
of up to 5 terms, and a split product at most 9 additions more.  The bound counts each as 2^-23 of A = |x| |W|
as if they all went one way: (5 n + 10) 2^-23 A; the smaller terms' instructions run over the same sum.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import mx_ref as R
from cogito_amd.capi import CGX_MX_FP4, CGX_MX_FP6, CGX_MX_FP32, DeviceArray, last_error
from gpu_util import device_tensor, host_tensor

pytestmark = pytest.mark.gpu
ACTS = [CGX_MX_FP4, CGX_MX_FP6, CGX_MX_FP32]


def _up(lib, a, t):
    return DeviceArray.from_numpy(lib, np.ascontiguousarray(a, t))


def _within(off, tol):
    """|off| <= tol everywhere (NaN nowhere), with a short message."""
    bad = ~(np.abs(off) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, by up to {np.nanmax(np.abs(off) / tol):.3g} times the bound, first at {np.argwhere(bad)[0]}"


def _ok(lib, rc):
    assert rc == 0 and lib.cgx_synchronize() == 0, last_error(lib)


def _rows(rng, n, K):
    x = rng.normal(size=(n, K)) * np.exp(rng.normal(size=K)) * np.exp(0.5 * rng.normal(size=(n, 1)))
    return x.astype(np.float32)


class Weight:
    def __init__(self, lib, codes, byte, K, N, grad=0, device=True):
        self.lib = lib
        self.keep = [_up(lib, codes, np.uint8), _up(lib, byte, np.uint8)] if device else \
            [np.ascontiguousarray(codes), np.ascontiguousarray(byte)]
        p = [a.ptr if device else a.ctypes.data for a in self.keep]
        self.ptr = lib.cgx_mx_weight_new(p[0], p[1], K, N, grad)
        assert self.ptr, last_error(lib)

    def __del__(self):
        if getattr(self, "ptr", None):
            self.lib.cgx_mx_weight_free(self.ptr)


# ------------------------------------------------------------ blocks

@pytest.mark.parametrize("fmt", [CGX_MX_FP4, CGX_MX_FP6])
@pytest.mark.parametrize("rows,cols,ld,off", [(1, 1, 1, 0), (3, 31, 31, 0), (5, 32, 32, 0), (7, 33, 40, 0), (2, 4096, 4096, 0),
                                              (67, 1000, 1003, 1), (4, 513, 516, 0), (130, 64, 64, 0)])
def test_quantise_and_read_back(gpu, fmt, rows, cols, ld, off):
    rng = np.random.default_rng(rows * cols)
    x = _rows(rng, rows, ld)
    t = R.TABLE[fmt]
    # ties, values next to them, the largest codes, zeros of both signs
    mid = np.concatenate([(t[1:] + t[:-1]) / 2, [t[-1] * 1.02, 7.9, 0.0, -0.0]]).astype(np.float32)
    mid = np.concatenate([mid, np.nextafter(mid, 9), np.nextafter(mid, -9)]).astype(np.float32)
    n = min(len(mid), ld)
    x[0, :n] = mid[:n] * rng.choice([-1, 1], n)
    if cols > 64:
        x[-1, 32:64] = 0
    buf = _up(gpu, np.concatenate([np.zeros(off, np.float32), x.ravel()]), np.float32)
    blocks = -(-cols // 32)
    size = 16 if fmt == CGX_MX_FP4 else 24
    codes, scales = _up(gpu, np.full(rows * blocks * size + 64, 0xA5), np.uint8), _up(gpu, np.full(rows * blocks + 64, 0xA5), np.uint8)
    y = _up(gpu, np.full(rows * ld + off + 16, 7.0), np.float32)
    _ok(gpu, gpu.cgx_mx_quantize_dev(buf.ptr + 4 * off, ld, rows, cols, fmt, codes.ptr, scales.ptr))
    _ok(gpu, gpu.cgx_mx_dequantize_dev(codes.ptr, scales.ptr, rows, cols, fmt, y.ptr + 4 * off, ld))
    q, b = R.quantise(x[:, :cols], fmt)
    got = codes.numpy(np.uint8, (codes.nbytes,))
    np.testing.assert_array_equal(scales.numpy(np.uint8, (rows * blocks + 64,))[:rows * blocks], b.ravel())
    np.testing.assert_array_equal(got[:rows * blocks * size], R.pack(q, fmt).ravel())
    assert np.all(got[rows * blocks * size:] == 0xA5)
    out = y.numpy(np.float32, (y.nbytes // 4,))
    full = out[off:off + rows * ld].reshape(rows, ld)
    np.testing.assert_array_equal(full[:, :cols], R.values(q, b, fmt, cols).astype(np.float32))
    assert np.all(full[:, cols:] == 7.0) and np.all(out[off + rows * ld:] == 7.0) and np.all(out[:off] == 7.0)


@pytest.mark.parametrize("fmt", [CGX_MX_FP4, CGX_MX_FP6])
def test_blocks_at_the_ends_of_the_range(gpu, fmt):
    rng = np.random.default_rng(3)
    with np.errstate(over="ignore"):
        x = np.concatenate([_rows(rng, 1, 32) * np.float32(s) for s in
                            (1e-45, 1e-40, 2.0 ** -126, 2.0 ** -124, 2.0 ** -120, 1e30, 3e37)])
    x[x == np.inf] = 3e38
    x = np.concatenate([x, np.full((1, 32), np.finfo(np.float32).max, np.float32), np.zeros((1, 32), np.float32)])
    special = np.ones((4, 32), np.float32)
    special[0, 3], special[1, 31], special[2, 0] = np.nan, np.inf, -np.inf
    x = np.concatenate([x, special]).astype(np.float32)
    n = len(x)
    d, codes, scales, y = _up(gpu, x, np.float32), DeviceArray(gpu, n * 24), DeviceArray(gpu, n), DeviceArray(gpu, n * 128)
    _ok(gpu, gpu.cgx_mx_quantize_dev(d.ptr, 32, n, 32, fmt, codes.ptr, scales.ptr))
    _ok(gpu, gpu.cgx_mx_dequantize_dev(codes.ptr, scales.ptr, n, 32, fmt, y.ptr, 32))
    q, b = R.quantise(x, fmt)
    np.testing.assert_array_equal(scales.numpy(np.uint8, (n,)), b[:, 0])
    got, exp = y.numpy(np.float32, (n, 32)), R.values(q, b, fmt, 32)
    np.testing.assert_array_equal(got[:-4], exp[:-4].astype(np.float32))
    assert np.all(np.isnan(got[-4:-1])) and np.all(got[-1] == 1)
    # any byte and code reads back
    raw = rng.integers(0, 256, (256, 24 if fmt == CGX_MX_FP6 else 16), dtype=np.uint8)
    by = np.arange(256, dtype=np.uint8)
    y, d_raw, d_by = DeviceArray(gpu, 256 * 128), _up(gpu, raw, np.uint8), _up(gpu, by, np.uint8)
    _ok(gpu, gpu.cgx_mx_dequantize_dev(d_raw.ptr, d_by.ptr, 256, 32, fmt, y.ptr, 32))
    exp = R.values(R.unpack(raw, 256, 1, fmt), by[:, None], fmt, 32)
    with np.errstate(over="ignore"):
        np.testing.assert_array_equal(y.numpy(np.float32, (256, 32)), exp.astype(np.float32))


# ----------------------------------------------------------- product

def _tol(x, xe, W, K, act):
    n = -(-K // 128)
    return ((5 if act == CGX_MX_FP32 else 1) * n + 10) * 2.0 ** -23 * (np.abs(x) @ np.abs(W)) + xe @ np.abs(W)


def _matmul(gpu, w, x, K, N, act, ldx=0, ldy=0, offx=0, offy=0):
    M = len(x)
    ldx, ldy = ldx or K, ldy or N
    buf = np.full((M, ldx), np.nan, np.float32)
    buf[:, :K] = x
    dx = _up(gpu, np.concatenate([np.zeros(offx, np.float32), buf.ravel()]), np.float32)
    y = _up(gpu, np.full(M * ldy + offy + 8, 7.0), np.float32)
    n = gpu.cgx_matmul_mx_ws(w.ptr, M, act)
    ws = _up(gpu, np.full(n + 256, 0xC3), np.uint8)
    _ok(gpu, gpu.cgx_matmul_mx_dev(dx.ptr + 4 * offx, ldx, M, w.ptr, act, y.ptr + 4 * offy, ldy, ws.ptr, n))
    assert np.all(ws.numpy(np.uint8, (n + 256,))[n:] == 0xC3)
    out = y.numpy(np.float32, (y.nbytes // 4,))
    full = out[offy:offy + M * ldy].reshape(M, ldy)
    assert np.all(full[:, N:] == 7.0) and np.all(out[offy + M * ldy:] == 7.0) and np.all(out[:offy] == 7.0)
    return full[:, :N].copy()


SHAPES = [(1, 1, 1), (1, 32, 16), (2, 33, 17), (5, 127, 255), (5, 128, 256), (16, 129, 257), (17, 512, 40), (31, 1000, 300), (33, 640, 511),
          (48, 96, 2401), (64, 256, 512), (65, 257, 130), (129, 300, 260), (200, 1024, 100), (1, 4096, 1000), (5, 11008, 64), (260, 11008, 33)]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_product(gpu, M, K, N, act):
    rng = np.random.default_rng(M * 7 + K * 3 + N)
    codes, byte, W = R.weight(rng, N, K, 0.05, 3)
    x = _rows(rng, M, K)
    w = Weight(gpu, codes, byte, K, N, device=M % 2 == 1)
    y = _matmul(gpu, w, x, K, N, act)
    xt = R.taken(x, act)
    _within(y - xt @ W, _tol(xt, R.cut_error(x, act), W, K, act))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [3, 40, 150])
def test_product_strides_and_alignment(gpu, M, act):
    rng = np.random.default_rng(M)
    K, N = 200, 301
    codes, byte, W = R.weight(rng, N, K)
    x = _rows(rng, M, K)
    w = Weight(gpu, codes, byte, K, N)
    first = _matmul(gpu, w, x, K, N, act)
    for ldx, ldy, ox, oy in ((201, 302, 0, 0), (204, 304, 0, 0), (208, 304, 1, 3), (200, 301, 2, 1)):
        np.testing.assert_array_equal(_matmul(gpu, w, x, K, N, act, ldx, ldy, ox, oy), first)


@pytest.mark.parametrize("act", ACTS)
def test_rows_do_not_depend_on_each_other(gpu, act):
    """A row with a NaN, an infinity or huge values leaves the others as they are; zeros and no rows."""
    rng = np.random.default_rng(5)
    K, N = 300, 70
    codes, byte, W = R.weight(rng, N, K)
    w = Weight(gpu, codes, byte, K, N)
    x = _rows(rng, 20, K)
    first = _matmul(gpu, w, x, K, N, act)
    z = x.copy()
    z[3, 299], z[7, 0], z[11], z[12] = np.nan, np.inf, 0, 1e30
    y = _matmul(gpu, w, z, K, N, act)
    assert np.all(np.isnan(y[[3, 7]])) and np.all(y[11] == 0) and np.all(np.isfinite(y[12]))
    keep = [i for i in range(20) if i not in (3, 7, 11, 12)]
    np.testing.assert_array_equal(y[keep], first[keep])
    assert gpu.cgx_matmul_mx_dev(w.keep[0].ptr, K, 0, w.ptr, act, w.keep[1].ptr, N, None, 0) == 0


@pytest.mark.parametrize("M", [2, 40])
@pytest.mark.parametrize("act", ACTS)
def test_nan_meets_zero(gpu, M, act):
    """A NaN of a row makes its output NaN where the weight is 0 too, and one of a weight's block where the row is 0."""
    K, N = 128, 40
    codes, byte, _ = R.weight(np.random.default_rng(7), N, K)
    codes[3] = 0
    byte[5, 2] = 255
    w = Weight(gpu, codes, byte, K, N)
    x = np.ones((M, K), np.float32)
    x[0, 70] = np.nan
    x[1] = 0
    y = _matmul(gpu, w, x, K, N, act)
    assert np.all(np.isnan(y[0])) and np.all(np.isnan(y[:, 5])) and np.all(np.isfinite(np.delete(y[1:], 5, 1)))


def test_weight_bytes_of_every_size(gpu):
    """Scales 0 to 254, blocks of byte 255, and rows of small and large values."""
    rng = np.random.default_rng(6)
    K, N = 64, 256
    codes, _, _ = R.weight(rng, N, K)
    byte = np.stack([np.arange(256), np.arange(256)], 1).astype(np.uint8)
    c = R.unpack(codes, N, 2, 4)
    w = Weight(gpu, codes, byte, K, N)
    W = R.values(c, byte, 4, K).T
    for size, lo, hi in ((1.0, 20, 250), (2.0 ** 100, 0, 140), (2.0 ** -90, 90, 254)):
        x = (rng.normal(size=(5, K)) * size).astype(np.float32)
        y = _matmul(gpu, w, x, K, N, CGX_MX_FP32)
        assert np.all(np.isnan(y[:, 255]))
        exp, tol = x.astype(np.float64) @ W[:, lo:hi], _tol(np.abs(x), R.cut_error(x, 32), W[:, lo:hi], K, CGX_MX_FP32)
        _within(y[:, lo:hi] - exp, tol + 1e-37)


def test_values_far_apart_in_a_row(gpu):
    """Blocks 2^60 apart each keep their bits: the weights of the large block are zero in every second column."""
    rng = np.random.default_rng(8)
    K, N = 256, 64
    w64 = rng.normal(size=(N, K))
    w64[::2, :32] = 0
    c, b = R.quantise(w64.astype(np.float32), 4)
    W = R.values(c, b, 4, K).T
    x = _rows(rng, 6, K)
    x[:, :32] *= np.float32(2.0 ** 60)
    w = Weight(gpu, R.pack(c, 4), b, K, N)
    y = _matmul(gpu, w, x, K, N, CGX_MX_FP32)
    tol = _tol(np.abs(x), R.cut_error(x, 32), W, K, CGX_MX_FP32)
    tol[:, ::2] = _tol(np.abs(x[:, 32:]), R.cut_error(x, 32)[:, 32:], W[32:, ::2], K, CGX_MX_FP32)
    _within(y - x.astype(np.float64) @ W, tol)


@pytest.mark.parametrize("device", [False, True])
@pytest.mark.parametrize("K,N", [(1, 1), (100, 33), (256, 512)])
def test_weight_of_a_tensor(gpu, K, N, device):
    """The same weight as that of its quantised transpose, bit for bit."""
    rng = np.random.default_rng(K)
    W = rng.normal(size=(K, N)).astype(np.float32)
    t = (device_tensor if device else host_tensor)(gpu, W)
    c, b = R.quantise(W.T, 4)
    a = Weight(gpu, R.pack(c, 4), b, K, N)
    h = gpu.cgx_mx_weight_from_tensor(t, 0)
    assert h, last_error(gpu)
    x = _rows(rng, 4, K)
    first = _matmul(gpu, a, x, K, N, CGX_MX_FP32)
    own, a.ptr = a.ptr, h
    np.testing.assert_array_equal(_matmul(gpu, a, x, K, N, CGX_MX_FP32), first)
    gpu.cgx_mx_weight_free(own)
    gpu.cg_tensor_free(t)


def test_more_rows_than_a_launch_takes(gpu):
    rng = np.random.default_rng(9)
    K, N, M = 40, 20, 4096 + 70
    codes, byte, W = R.weight(rng, N, K)
    x = _rows(rng, M, K)
    y = _matmul(gpu, Weight(gpu, codes, byte, K, N), x, K, N, CGX_MX_FP32)
    _within(y - x.astype(np.float64) @ W, _tol(np.abs(x), R.cut_error(x, 32), W, K, CGX_MX_FP32))


# -------------------------------------------------------------- loss

class Loss:
    """Buffers of a call; guard words behind every output."""

    def __init__(self, gpu, w, h, targets, act, V, dloss=None, ldh=0, ldd=0, grad=True):
        self.gpu, self.w, self.act, self.n, self.K = gpu, w, act, len(h), h.shape[1]
        self.ldh, self.ldd, self.grad = ldh or self.K, ldd or self.K, grad
        buf = np.full((self.n, self.ldh), np.nan, np.float32)
        buf[:, :self.K] = h
        self.h, self.t = _up(gpu, buf, np.float32), _up(gpu, targets, np.int32)
        self.g = None if dloss is None else _up(gpu, dloss, np.float32)
        self.loss, self.lse = (_up(gpu, np.full(self.n + 4, 7.0), np.float32) for _ in range(2))
        self.dh = _up(gpu, np.full(self.n * self.ldd + 4, 7.0), np.float32)
        self.need = gpu.cgx_token_loss_mx_ws(w.ptr, self.n, act, int(grad))
        self.ws = _up(gpu, np.full(self.need + 256, 0xC3), np.uint8)

    def forward(self):
        return self.gpu.cgx_token_loss_mx_dev(self.h.ptr, self.ldh, self.n, self.w.ptr, self.act, self.t.ptr,
                                              self.loss.ptr, self.lse.ptr, self.ws.ptr, self.need)

    def backward(self):
        return self.gpu.cgx_token_loss_mx_grad_dev(self.h.ptr, self.ldh, self.n, self.w.ptr, self.act, self.t.ptr, self.lse.ptr,
                                                   self.g.ptr if self.g else None, self.dh.ptr, self.ldd, self.ws.ptr, self.need)

    def run(self):
        _ok(self.gpu, self.forward())
        if self.grad:
            _ok(self.gpu, self.backward())
        return self.read()

    def read(self):
        assert np.all(self.ws.numpy(np.uint8, (self.need + 256,))[self.need:] == 0xC3)
        a, b, d = (x.numpy(np.float32, (x.nbytes // 4,)) for x in (self.loss, self.lse, self.dh))
        assert np.all(a[self.n:] == 7) and np.all(b[self.n:] == 7) and np.all(d[self.n * self.ldd:] == 7)
        d = d[:self.n * self.ldd].reshape(self.n, self.ldd)
        assert np.all(d[:, self.K:] == 7)
        return a[:self.n], b[:self.n], d[:, :self.K].copy()


def _check(out, h, W, targets, act, dloss=None, grad=True):
    """Bounds: a logit is off by at most T (the product's); lse by max T, 2^-22 for the fp32 exponentials and sums (each of
    exp's 2 ulp, the sums of 128 values a wave in 32 bits: 128 2^-24 = 2^-17 if all went one way; parts in 64) and its own
    rounding; p = exp(z - lse) by a factor of 1 + 2 max T + 2^-20 + 2^-22 |lse|; its records hold 2^-23 of a block's largest, at
    most 1; the second product's sums as the first's over chunks of the vocabulary, and additions of the pieces."""
    lse, loss, dh, z = R.loss(h, W, targets, act, dloss)
    x, K, V = R.taken(h, act), W.shape[0], W.shape[1]
    T = _tol(np.abs(x), R.cut_error(h, act), W, K, act).max(1)
    e = T + 2.0 ** -17 + 2.0 ** -23 * np.abs(lse)
    _within(out[1] - lse, e)
    _within(out[0] - loss, e + T + 2.0 ** -23 * np.abs(loss))
    if not grad:
        return
    live = (np.asarray(targets) >= 0) & (np.asarray(targets) < V)
    p = np.exp(z - lse[:, None])
    q = p.copy()
    q[np.arange(len(z))[live], np.asarray(targets)[live]] -= 1
    A = np.abs(W).T
    near = p * (e + T + 2.0 ** -20)[:, None]
    block = np.pad(np.abs(q), ((0, 0), (0, -V % 32))).reshape(len(z), -1, 32).max(2)
    held = np.repeat(block * 2.0 ** -23, 32, 1)[:, :V]
    n = -(-V // 128)
    tol = (near + held) @ A + (5 * n + 20) * 2.0 ** -23 * (np.abs(q) @ A)
    g = np.where(live, 1.0 if dloss is None else np.abs(np.asarray(dloss, np.float64)), 0.0)
    _within(out[2] - dh, g[:, None] * tol + 1e-37)


def _targets(rng, n, V):
    t = rng.integers(0, V, n)
    t[n // 2] = V - 1
    if n > 2:
        t[0], t[n - 1] = 0, -1
    if n > 3:
        t[1] = V
    return t.astype(np.int32)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows,K,V", [(1, 1, 1), (1, 32, 100), (5, 128, 257), (16, 200, 4000), (17, 96, 130), (40, 300, 1000), (64, 64, 511), (70, 513, 640),
                                      (130, 128, 2500), (300, 40, 129)])
def test_loss_and_gradient(gpu, rows, K, V, act):
    rng = np.random.default_rng(rows + K + V)
    codes, byte, W = R.weight(rng, V, K, 1.5 / np.sqrt(K))
    h = _rows(rng, rows, K)
    t = _targets(rng, rows, V)
    g = rng.normal(size=rows).astype(np.float32)
    c = Loss(gpu, Weight(gpu, codes, byte, K, V, grad=1), h, t, act, V, g, ldh=K + 3, ldd=K + 1)
    out = c.run()
    _check(out, h, W, t, act, g)
    ignored = (t < 0) | (t >= V)
    assert np.all(out[0][ignored] == 0) and np.all(out[2][ignored] == 0)


@pytest.mark.parametrize("spread", [0, 4, 7, 30, 200])
def test_gradient_of_rows_far_apart(gpu, spread):
    """Vocabulary rows of sizes up to 2^spread apart within a block: further layers of the transposed weight."""
    rng = np.random.default_rng(spread)
    rows, K, V = 9, 70, 700
    w64 = rng.normal(size=(V, K))
    w64[200:400] *= np.exp2(-rng.integers(0, spread + 1, (200, 1)).astype(np.float64))
    c, b = R.quantise(w64.astype(np.float32), 4)
    W = R.values(c, b, 4, K).T
    h = _rows(rng, rows, K) * np.float32(0.3)
    # targets among the smallest rows, and a gradient that is theirs alone in some inputs
    t = rng.integers(200, 400, rows).astype(np.int32)
    out = Loss(gpu, Weight(gpu, R.pack(c, 4), b, K, V, grad=1), h, t, CGX_MX_FP32, V).run()
    _check(out, h, W, t, CGX_MX_FP32)


def test_gradient_against_differences(gpu):
    """Central differences of the 64-bit loss in random directions, step 1e-4: their error is O(step^2), below 1e-6 here."""
    rng = np.random.default_rng(12)
    rows, K, V = 6, 64, 300
    codes, byte, W = R.weight(rng, V, K, 0.2)
    h = rng.normal(size=(rows, K)).astype(np.float32)
    t = rng.integers(0, V, rows).astype(np.int32)
    dh = Loss(gpu, Weight(gpu, codes, byte, K, V, grad=1), h, t, CGX_MX_FP32, V).run()[2]
    for _ in range(4):
        d = rng.normal(size=(rows, K))
        f = [R.loss(h + s * 1e-4 * d, W, t, 32)[1] for s in (1, -1)]
        np.testing.assert_allclose((dh * d).sum(1), (f[0] - f[1]) / 2e-4, atol=2e-5)


def test_loss_of_extreme_rows(gpu):
    rng = np.random.default_rng(13)
    K, V = 64, 400
    codes, byte, W = R.weight(rng, V, K, 1.0)
    h = _rows(rng, 8, K)
    h[1] = 0                                           # uniform
    h[2] *= 300                                        # one token has all the mass
    h[3, 5], h[4, 63] = np.nan, np.inf
    h[5] *= np.float32(1e-30)
    t = _targets(rng, 8, V)
    t[:] = rng.integers(0, V, 8)
    t[7] = -1
    h[7, 0] = np.nan                                   # an ignored row
    t[2] = int((h[2].astype(np.float64) @ W).argmax())
    loss, lse, dh = Loss(gpu, Weight(gpu, codes, byte, K, V, grad=1), h, t, CGX_MX_FP32, V).run()
    assert np.all(np.isnan(lse[[3, 4, 7]])) and np.all(np.isnan(loss[[3, 4]])) and np.all(np.isnan(dh[[3, 4]]))
    assert loss[7] == 0 and np.all(dh[7] == 0)
    ok = [0, 1, 2, 5, 6]
    _check((loss[ok], lse[ok], dh[ok]), h[ok], W, t[ok], CGX_MX_FP32)


def test_loss_outputs_left_out(gpu):
    rng = np.random.default_rng(14)
    K, V, n = 96, 300, 5
    codes, byte, W = R.weight(rng, V, K)
    w = Weight(gpu, codes, byte, K, V)
    c = Loss(gpu, w, _rows(rng, n, K), _targets(rng, n, V), CGX_MX_FP32, V, grad=False)
    both = c.run()
    for a, b in ((c.loss.ptr, None), (None, c.lse.ptr)):
        c.loss.upload(np.full(n + 4, 7, np.float32))
        c.lse.upload(np.full(n + 4, 7, np.float32))
        _ok(gpu, gpu.cgx_token_loss_mx_dev(c.h.ptr, K, n, w.ptr, CGX_MX_FP32, c.t.ptr, a, b, c.ws.ptr, c.need))
        got = c.read()
        np.testing.assert_array_equal(got[0], both[0] if a else np.full(n, 7, np.float32))
        np.testing.assert_array_equal(got[1], both[1] if b else np.full(n, 7, np.float32))
    assert gpu.cgx_token_loss_mx_grad_dev(c.h.ptr, K, n, w.ptr, CGX_MX_FP32, c.t.ptr, c.lse.ptr, None, c.dh.ptr, K,
                                          c.ws.ptr, c.need) == -1
    assert "without a gradient" in last_error(gpu)


def test_nan_in_the_weight(gpu):
    rng = np.random.default_rng(15)
    K, V, n = 128, 300, 5
    codes, byte, _ = R.weight(rng, V, K)
    byte[17, 1] = 255
    c = Loss(gpu, Weight(gpu, codes, byte, K, V, grad=1), _rows(rng, n, K), np.array([1, 2, 3, 17, -1], np.int32), CGX_MX_FP32, V)
    loss, lse, dh = c.run()
    assert np.all(np.isnan(lse)) and np.all(np.isnan(loss[:4])) and np.all(np.isnan(dh[:4]))
    assert loss[4] == 0 and np.all(dh[4] == 0)
