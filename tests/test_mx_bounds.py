"""CPU: the ends of the ranges that the microscaled entry points allow.  Sizes that pass are told by the refusal that comes
next (a misaligned argument), so that no call here gets as far as a launch, with a device or without."""
from __future__ import annotations

import ctypes as C

import pytest

from cogito_amd.capi import CGX_MX_FP4, CGX_MX_FP6, CGX_MX_FP32, last_error
from test_mx_api import Weight

FAR = 1 << 44                                                # never read: the calls are refused first


def _refused(lib, rc, word):
    assert rc == -1 and word in last_error(lib), last_error(lib)
    lib.cgx_clear_error()


@pytest.fixture(autouse=True)
def _clear(lib):
    lib.cgx_clear_error()


@pytest.mark.parametrize("fmt", [CGX_MX_FP4, CGX_MX_FP6])
@pytest.mark.parametrize("name", ["cgx_mx_quantize_dev", "cgx_mx_dequantize_dev"])
def test_most_blocks_of_a_launch(lib, name, fmt):
    """A wave takes 512 values of a row and a block four waves of 64 lanes: 2^26 - 4 waves are 2^32 - 256 threads, one more
    is a block more, 2^32 threads, which a launch cannot have."""
    def call(rows, cols, codes):
        if name == "cgx_mx_quantize_dev":
            return lib.cgx_mx_quantize_dev(2 * FAR, cols, rows, cols, fmt, codes, 3 * FAR)
        return lib.cgx_mx_dequantize_dev(codes, 3 * FAR, rows, cols, fmt, 2 * FAR, cols)
    top = (1 << 26) - 4
    for rows, cols in ((top, 1), (top, 512), (top // 2, 513), (top // 4, 2048)):
        _refused(lib, call(rows, cols, FAR + 8), "aligned")
    for rows, cols in ((top + 1, 1), (top + 1, 512), (top + 2, 32), (top + 3, 1), (top // 2 + 1, 513), (top // 4 + 1, 2048)):
        _refused(lib, call(rows, cols, FAR + 8), "are required")


@pytest.mark.parametrize("off", [1, 2, 3])
def test_misaligned_arrays_of_a_loss(lib, off):
    """One part of a call reads a row's target by scalar loads, which leave an address' low bits out, others by vector loads:
    a misaligned array would give them different targets."""
    w = Weight.of(100, 600)
    n = lib.cgx_token_loss_mx_ws(C.byref(w), 4, CGX_MX_FP32, 1)

    def forward(targets=3 * FAR, loss=4 * FAR, lse=5 * FAR):
        return lib.cgx_token_loss_mx_dev(2 * FAR, 100, 4, C.byref(w), CGX_MX_FP32, targets, loss, lse, FAR, n)

    def gradient(targets=3 * FAR, lse=5 * FAR, dloss=6 * FAR):
        return lib.cgx_token_loss_mx_grad_dev(2 * FAR, 100, 4, C.byref(w), CGX_MX_FP32, targets, lse, dloss, 7 * FAR, 100, FAR, n)
    for call, names in ((forward, ("targets", "loss", "lse")), (gradient, ("targets", "lse", "dloss"))):
        for name in names:
            at = dict(targets=3, loss=4, lse=5, dloss=6)[name] * FAR
            _refused(lib, call(**{name: at + off}), "4-byte aligned")
