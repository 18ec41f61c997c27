"""CPU: the shapes of the GPU tests of microscaled products reach the forms that they stand for (told by the workspaces that the
library asks for), and a cut with a term less would not pass those tests."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import mx_cut as X
import mx_forms as F
import mx_ref as R
from cogito_amd.capi import CGX_MX_FP4, CGX_MX_FP6, CGX_MX_FP32
from test_mx_api import ACTS, Weight


def _whole(n):
    return (n + 255) & ~255


@pytest.fixture(autouse=True)
def _sizes(lib):
    lib.cgk_mx_matmul_need.restype = lib.cgk_mx_loss_need.restype = C.c_size_t


def _few(lib, M, K, N, act=CGX_MX_FP32):
    """Whether rows take the kernel of few rows, which needs no workspace."""
    return lib.cgk_mx_matmul_need(C.byref(Weight.of(K, N)), M, act) == 0


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("N,tiles", F.TILES)
def test_tiles_of_a_block(lib, N, tiles, act):
    """The loss of few rows keeps 8 bytes a row and group of `tiles` tiles, and 4 a row."""
    for M in F.FEW:
        assert _few(lib, M, 200, N, act)
        groups = -(-(-(-N // 16)) // tiles)
        assert lib.cgk_mx_loss_need(C.byref(Weight.of(200, N)), M, act, 0) == _whole(8 * M * groups) + _whole(4 * M)


def test_segments(lib):
    """Five terms of 24 bytes and a scale, four blocks a chunk, an odd number of chunks a row, against 152 KiB of LDS."""
    for M, K, N in F.SEGMENTS:
        assert _few(lib, M, K, N)
        assert M * (-(-K // 128) | 1) * 4 * (5 * 24 + 1) > 152 << 10
    assert sum(-(-N // 16) > 256 * 8 for _, _, N in F.SEGMENTS) >= 2


def test_borders_and_blocks(lib):
    for a, b in F.BORDERS:
        assert _few(lib, *a) and not _few(lib, *b), (a, b)
    for s in F.BLOCKS:
        assert not _few(lib, *s), s


def test_five_terms_hold_a_value():
    """The block's largest is 4 to 8 units of its scale.  A first term in steps of 1/2 from 4 units on leaves 1/4, or up to 1/2 from
    7.75 on, where it saturates at 7.5; of the second's units, 1/8 of the first's, that is 2, or 4, whose term in steps of 1/8, or
    1/4, leaves 1/16, or 1/8; of the third's, 1/32 of the second's, 2 and 4 again, and so on.  Four terms leave 2^-4 2^-13 of 4
    units, 2^-19, or 2^-3 2^-13 of 7.75, 32/31 2^-19; five 32/31 2^-24 (2^-23 is what the interface states)."""
    rng = np.random.default_rng(41)
    x = (rng.normal(size=(200, 320)) * np.exp(4 * rng.normal(size=(200, 320)))).astype(np.float32)
    off = np.abs(X.cut(x) - x).reshape(200, -1, 32).max(2) / np.abs(x).reshape(200, -1, 32).max(2)
    assert off.max() <= 32 / 31 * 2.0 ** -24
    four = np.abs(X.cut(x, 4) - x).reshape(200, -1, 32).max(2) / np.abs(x).reshape(200, -1, 32).max(2)
    assert 32 / 31 * 2.0 ** -19 >= four.max() > 2.0 ** -19.5


@pytest.mark.parametrize("M,K,N", F.SEGMENTS + F.BLOCKS + [(M, 200, N) for N, _ in F.TILES for M in F.FEW])
def test_a_term_less_would_show_in_a_product(M, K, N):
    x, _, _, _ = X.one_value_rows(M, K, 8, reps=-(-24 // M))
    alone = np.zeros((x.size, 32), np.float32)
    alone[:, 3] = x.ravel()
    off = lambda n: np.abs(X.cut(alone, n) - alone)[:, 3] / x.ravel()  # noqa: E731
    assert off(5).max() <= 2.0 ** -23
    # the right result is within 6 2^-23, so that a wrong one shows from twice that on
    assert np.all(off(4) > 2 * X.ONE_VALUE) and np.all(off(3) > 2 * X.ONE_VALUE)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,K,V", [(5, 700, 700), (20, 2100, 2100), (40, 96, 3000)])
def test_a_term_less_would_show_in_a_gradient(M, K, V, act):
    _, of, _, _, _, _, tol, q = X.one_output_inputs(M, K, V, lambda h: R.taken(h, act))
    off = lambda n: np.abs(X.cut(q, n) - q)[:, of]  # noqa: E731
    assert np.all(off(5) <= tol)
    assert (off(4) > 2 * tol).mean() > 0.02 and (off(3) > 2 * tol).mean() > 0.5
