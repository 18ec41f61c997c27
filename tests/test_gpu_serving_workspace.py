"""GPU: one workspace, sized for the largest call, under smaller ones.  Tolerance of the attention: that of
test_gpu_paged.py, 8e-6 of sum_j p_j |v_j| and the fixed-point term of the weights."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from cogito_amd.capi import CgxPagedStep, DeviceArray, last_error

pytestmark = pytest.mark.gpu
TOL = 8e-6


def _up(lib, a, t=np.int32):
    return DeviceArray.from_numpy(lib, np.ascontiguousarray(a, t))


@pytest.mark.parametrize("H,Hk,D,gs", [(8, 2, 128, 128), (12, 12, 64, 32), (8, 8, 256, 256)])
def test_attention_of_a_batch_that_drains(gpu, H, Hk, D, gs):
    """The batch's first sequences alone, down to one row, in the workspace of the whole batch."""
    rng = np.random.default_rng(D + H)
    b = R.Batch(gpu, rng, [1500, 900, 40, 700, 77, 1300], [1, 9, 40, 2, 4, 10], 16, H, Hk, D, gs).bind()
    n = gpu.cgx_attention_paged_ws(C.byref(b.cache), C.byref(b.step), H)
    O, _, A, F = b.reference()
    for seqs in (6, 5, 3, 2, 1):
        rows = int(b.begin[seqs])
        for most in (0, max(b.rows[:seqs])):
            st = CgxPagedStep(seqs=seqs, rows=rows, max_rows=most, table_ld=b.step.table_ld)
            st.table, st.row_begin, st.row_seq, st.kv_len = b.step.table, b.step.row_begin, b.step.row_seq, b.step.kv_len
            assert gpu.cgx_attention_paged_ws(C.byref(b.cache), C.byref(st), H) <= n
            ws = _up(gpu, np.full(n + 256, 0xC3), np.uint8)          # guard words behind the size asked for
            o = _up(gpu, np.full((b.T, H, D), 7.0), np.float32)
            assert gpu.cgx_attention_paged_dev(C.byref(b.cache), 0, C.byref(st), b.d["q"].ptr, H, None, None, o.ptr, None,
                                               ws.ptr, n) == 0, last_error(gpu)
            assert gpu.cgx_synchronize() == 0, last_error(gpu)
            assert np.all(ws.numpy(np.uint8, (n + 256,))[n:] == 0xC3)
            got = o.numpy(np.float32, (b.T, H, D))
            assert np.all(np.abs(got[:rows] - O[:rows]) <= TOL * A[:rows] + F[:rows] + 1e-37), (seqs, most)
            assert np.all(got[rows:] == 7.0)


def test_logprobs_of_a_batch_that_drains(gpu):
    """256 rows of 32000 take longer segments than 255 and fewer: the same numbers from the same workspace."""
    rng = np.random.default_rng(1)
    V, n_top, most = 32000, 20, 256
    x, tok = rng.normal(size=(most, V)).astype(np.float32), rng.integers(0, V, most)
    n = gpu.cgx_token_logprobs_ws(most, V, n_top)
    dx, dt, ws = _up(gpu, x, np.float32), _up(gpu, tok), _up(gpu, np.full(n + 256, 0xC3), np.uint8)
    order = np.argsort(-x, 1, kind="stable")[:, :n_top]
    lse = np.log(np.exp(x.astype(np.float64)).sum(1))
    for rows in (256, 255, 100, 1):
        lp, rank, ent, top, top_lp = (_up(gpu, np.full(rows * k + 4, -77)) for k in (1, 1, 1, n_top, n_top))
        assert gpu.cgx_token_logprobs_dev(dx.ptr, V, rows, V, dt.ptr, n_top, lp.ptr, rank.ptr, ent.ptr, top.ptr,
                                          top_lp.ptr, ws.ptr, n) == 0, last_error(gpu)
        assert gpu.cgx_synchronize() == 0, last_error(gpu)
        assert np.all(ws.numpy(np.uint8, (n + 256,))[n:] == 0xC3)
        np.testing.assert_array_equal(top.numpy(np.int32, (rows * n_top + 4,))[:-4].reshape(rows, n_top), order[:rows])
        exp = x[np.arange(rows), tok[:rows]] - lse[:rows]
        # test_gpu_logprobs.py's bound of a log probability
        assert np.all(np.abs(lp.numpy(np.float32, (rows + 4,))[:rows] - exp) <= 6e-6 + np.abs(exp) * 2.0 ** -23)
        assert np.all(lp.numpy(np.int32, (rows + 4,))[rows:] == -77)
