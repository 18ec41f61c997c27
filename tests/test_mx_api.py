"""CPU: what the microscaled entry points refuse, and their workspaces' sizes.  Calls that pass every check fail
here for want of a device, so each refusal is told by its message."""
from __future__ import annotations

import ctypes as C

import pytest

from cogito_amd.capi import CGX_MX_FP4, CGX_MX_FP6, CGX_MX_FP32, last_error

_BUF = C.create_string_buffer(1 << 16)
P = (C.addressof(_BUF) + 15) & ~15                           # never read: the calls are refused first
FAR = P + (1 << 40)                                          # apart from it
ACTS = [CGX_MX_FP4, CGX_MX_FP6, CGX_MX_FP32]


class Weight(C.Structure):
    """The library's handle (cgx_internal.h), made without a device."""
    _fields_ = [("K", C.c_int), ("N", C.c_int), ("codes", C.c_void_p), ("chunks128", C.c_int), ("tcodes", C.c_void_p),
                ("list", C.c_void_p), ("first", C.POINTER(C.c_int)), ("tchunks", C.c_int)]

    @classmethod
    def of(cls, K, N, grad=1, layers=1):
        n = -(-N // 128)
        w = cls(K=K, N=N, codes=P, chunks128=n, tchunks=n * layers)
        if grad:
            w.tcodes, w.list = P, P
            w.first = (C.c_int * (n + 1))(*(i * layers for i in range(n + 1)))
        return w


def _refused(lib, rc, word):
    assert not rc or rc == -1
    assert word in last_error(lib), last_error(lib)
    lib.cgx_clear_error()


@pytest.fixture(autouse=True)
def _clear(lib):
    lib.cgx_clear_error()


@pytest.mark.parametrize("name", ["cgx_mx_quantize_dev", "cgx_mx_dequantize_dev"])
def test_blocks(lib, name):
    def call(x=FAR, ld=64, rows=4, cols=64, fmt=CGX_MX_FP4, codes=P, scales=P + 4096):
        if name == "cgx_mx_quantize_dev":
            return lib.cgx_mx_quantize_dev(x, ld, rows, cols, fmt, codes, scales)
        return lib.cgx_mx_dequantize_dev(codes, scales, rows, cols, fmt, x, ld)
    for kw in (dict(x=None), dict(codes=None), dict(scales=None), dict(rows=-1), dict(cols=0), dict(cols=-5), dict(ld=63), dict(ld=0),
               dict(fmt=CGX_MX_FP32), dict(fmt=0), dict(fmt=8), dict(rows=1 << 26), dict(rows=1 << 24, cols=4096, ld=4096),
               dict(ld=1 << 32), dict(rows=1, cols=(1 << 30) + 1, ld=(1 << 30) + 1)):
        _refused(lib, call(**kw), "are required")
    for kw in (dict(codes=P + 8), dict(x=FAR + 2)):
        _refused(lib, call(**kw), "aligned")
    out = dict(x=P + 16) if name == "cgx_mx_dequantize_dev" else dict(scales=P + 127)
    _refused(lib, call(**out), "overlaps")
    _refused(lib, call(x=P + 4096 - 4 * (3 * 64 + 64) + 4), "overlaps")
    # 6-bit codes are half as long again
    assert call(fmt=CGX_MX_FP6, rows=0, x=P) in (0, -1)


def test_weights(lib):
    for K, N in ((0, 5), (5, 0), (-1, 5), ((1 << 20) + 1, 1), (1, (1 << 24) + 1), (1 << 20, 1 << 17)):
        _refused(lib, lib.cgx_mx_weight_new(P, P, K, N, 0), "together at most")
    _refused(lib, lib.cgx_mx_weight_new(None, P, 5, 5, 0), "codes and scales")
    _refused(lib, lib.cgx_mx_weight_new(P, None, 5, 5, 0), "codes and scales")
    _refused(lib, lib.cgx_mx_weight_from_tensor(None, 0), "a matrix")
    t = lib.cg_tensor_full((C.c_int * 1)(4), 1, 1.0, False)
    _refused(lib, lib.cgx_mx_weight_from_tensor(t, 0), "a matrix")
    lib.cg_tensor_free(t)
    lib.cgx_mx_weight_free(None)


@pytest.mark.parametrize("act", ACTS)
def test_product(lib, act):
    w = Weight.of(100, 60)
    n = lib.cgx_matmul_mx_ws(C.byref(w), 4, act)

    def call(x=FAR, ldx=100, M=4, h=C.byref(w), a=act, y=2 * FAR, ldy=60, ws=P, size=n):
        return lib.cgx_matmul_mx_dev(x, ldx, M, h, a, y, ldy, ws, size)
    for kw in (dict(h=None), dict(M=-1), dict(M=1 << 23), dict(a=0), dict(a=8)):
        _refused(lib, call(**kw), "a weight")
    for kw in (dict(x=None), dict(y=None), dict(ldx=99), dict(ldy=59), dict(x=FAR + 1), dict(y=FAR + 2), dict(ldx=1 << 32), dict(ldy=1 << 32)):
        _refused(lib, call(**kw), "rows of")
    if n:
        for kw in (dict(ws=None), dict(ws=P + 8), dict(size=n - 1), dict(size=0)):
            _refused(lib, call(**kw), "workspace of")
        _refused(lib, call(x=P), "overlaps")
        _refused(lib, call(y=P), "overlaps")
    _refused(lib, call(y=FAR + 4 * 399), "overlaps")
    _refused(lib, lib.cgx_matmul_mx_ws(None, 4, act), "a weight")
    _refused(lib, lib.cgx_matmul_mx_ws(C.byref(w), 4, 5), "a weight")
    assert lib.cgx_matmul_mx_ws(C.byref(w), 0, act) == 0


@pytest.mark.parametrize("act", ACTS)
def test_loss(lib, act):
    w, plain = Weight.of(100, 600), Weight.of(100, 600, grad=0)
    n = lib.cgx_token_loss_mx_ws(C.byref(w), 4, act, 1)
    assert lib.cgx_token_loss_mx_ws(C.byref(w), 4, act, 0) <= n

    def call(h=FAR, ld=100, rows=4, w_=C.byref(w), a=act, t=3 * FAR, loss=4 * FAR, lse=5 * FAR, ws=P, size=n):
        return lib.cgx_token_loss_mx_dev(h, ld, rows, w_, a, t, loss, lse, ws, size)

    def grad(h=FAR, ld=100, rows=4, w_=C.byref(w), a=act, t=3 * FAR, lse=5 * FAR, g=6 * FAR, dh=7 * FAR, ldd=100, ws=P, size=n):
        return lib.cgx_token_loss_mx_grad_dev(h, ld, rows, w_, a, t, lse, g, dh, ldd, ws, size)
    for f in (call, grad):
        for kw in (dict(w_=None), dict(rows=-1), dict(rows=1 << 23), dict(a=1)):
            _refused(lib, f(**kw), "a weight")
        for kw in (dict(h=None), dict(ld=99), dict(h=FAR + 2), dict(ld=1 << 32)):
            _refused(lib, f(**kw), "rows of")
        for kw in (dict(ws=None), dict(ws=P + 4), dict(size=0)):
            _refused(lib, f(**kw), "workspace of")
        _refused(lib, f(t=None), "targets")
        for kw in (dict(h=P), dict(t=P), dict(lse=P), dict(lse=P + 64)):
            _refused(lib, f(**kw), "overlaps")
    _refused(lib, call(loss=None, lse=None), "loss or lse")
    _refused(lib, call(loss=5 * FAR + 12), "overlaps")
    _refused(lib, call(loss=3 * FAR), "overlaps")
    _refused(lib, grad(lse=None), "lse")
    for kw in (dict(dh=None), dict(ldd=99), dict(dh=FAR + 3)):
        _refused(lib, grad(**kw), "rows of")
    for kw in (dict(dh=FAR), dict(dh=5 * FAR), dict(dh=6 * FAR - 4), dict(g=P)):
        _refused(lib, grad(**kw), "overlaps")
    _refused(lib, grad(w_=C.byref(plain)), "without a gradient")
    _refused(lib, lib.cgx_token_loss_mx_ws(C.byref(plain), 4, act, 1), "without a gradient")
    assert lib.cgx_token_loss_mx_ws(C.byref(w), 0, act, 1) == 0


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("K,N", [(1, 1), (96, 70), (768, 50257), (4096, 4096), (11008, 4096), (4096, 22016), (4096, 128256), (40, 1000000)])
@pytest.mark.parametrize("layers", [1, 3])
def test_workspaces_grow_with_the_call(lib, act, K, N, layers):
    """A size is enough for every call of fewer rows: no call of m rows refuses the size of M >= m."""
    w = Weight.of(K, N, layers=layers)
    lib.cgk_mx_matmul_need.restype = lib.cgk_mx_loss_need.restype = C.c_size_t
    rows = sorted({r + d for r in (1, 16, 32, 48, 64, 100, 128, 256, 300, 512, 1000, 2048, 4096, 6000, 8192, 70000) for d in (-1, 0, 1)} - {0})
    sizes = [[lib.cgx_matmul_mx_ws(C.byref(w), r, act) for r in rows]] + \
            [[lib.cgx_token_loss_mx_ws(C.byref(w), r, act, g) for r in rows] for g in (0, 1)]
    assert last_error(lib) == ""
    for s in sizes:
        assert s == sorted(s)
    for i, r in enumerate(rows):
        assert lib.cgk_mx_matmul_need(C.byref(w), r, act) <= sizes[0][i]
        for g in (0, 1):
            assert lib.cgk_mx_loss_need(C.byref(w), r, act, g) <= sizes[1 + g][i]
