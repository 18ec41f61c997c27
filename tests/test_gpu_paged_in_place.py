"""GPU: the calls of a serving step that may write over what they read give the bits of the ones that do not."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from cogito_amd.capi import CgxPagedStep, DeviceArray, last_error

pytestmark = pytest.mark.gpu


def _up(lib, a, t=np.float32):
    return DeviceArray.from_numpy(lib, np.ascontiguousarray(a, t))


@pytest.mark.parametrize("H,Hk,D,gs", [(32, 8, 128, 128), (12, 12, 64, 32), (4, 2, 256, 256), (16, 1, 64, 16)])
@pytest.mark.parametrize("kv,rows", [([40], [1]), ([3000, 700, 20, 1200], [5, 40, 3, 9]), ([300], [130])])
def test_attention_over_its_queries(gpu, H, Hk, D, gs, kv, rows):
    b = R.Batch(gpu, np.random.default_rng(D + sum(kv)), kv, rows, 16, H, Hk, D, gs, pad=2).bind()
    o, ls = b.attend()
    n = gpu.cgx_attention_paged_ws(C.byref(b.cache), C.byref(b.step), H)
    ws, q, lse = DeviceArray(gpu, max(n, 16)), _up(gpu, b.q), _up(gpu, np.zeros((b.T, H)))
    assert gpu.cgx_attention_paged_dev(C.byref(b.cache), 0, C.byref(b.step), q.ptr, H, None, None, q.ptr, lse.ptr, ws.ptr, n) == 0
    assert gpu.cgx_synchronize() == 0, last_error(gpu)
    m = int(b.begin[-1])
    got = q.numpy(np.float32, (b.T, H, D))
    np.testing.assert_array_equal(got[:m], o[:m])
    np.testing.assert_array_equal(got[m:], b.q[m:])
    np.testing.assert_array_equal(lse.numpy(np.float32, (b.T, H))[:m], ls[:m])


@pytest.mark.parametrize("H,Hk,D,gs", [(32, 8, 128, 128), (7, 9, 256, 2), (3, 1, 96, 32)])
def test_append_of_one_row_in_its_place(gpu, H, Hk, D, gs):
    rng = np.random.default_rng(H)
    x, cs = rng.normal(size=(1, (H + 2 * Hk) * D)).astype(np.float32), rng.normal(size=(9, D // 2, 2)).astype(np.float32)
    got = []
    for in_place in (False, True):
        pool = R.Pool(1, 2, 16, Hk, D, gs)
        cache = pool.upload(gpu)
        dx, dcs, q = _up(gpu, x), _up(gpu, cs), _up(gpu, np.zeros((H, D)))
        slot, pos = _up(gpu, [19], np.int32), _up(gpu, [8], np.int32)
        st = CgxPagedStep(seqs=1, rows=1, max_rows=0, table_ld=1)
        st.row_slot, st.row_pos = slot.ptr, pos.ptr
        assert gpu.cgx_kv_paged_append_dev(C.byref(cache), 0, C.byref(st), dx.ptr, x.shape[1], H, dcs.ptr, 9,
                                           (dx if in_place else q).ptr) == 0, last_error(gpu)
        assert gpu.cgx_synchronize() == 0, last_error(gpu)
        after = dx.numpy(np.float32, x.shape)[0]
        np.testing.assert_array_equal(after[H * D:], x[0, H * D:])
        got.append([after[:H * D] if in_place else q.numpy(np.float32, (H * D,))] + pool.download())
    for a, b in zip(*got):
        np.testing.assert_array_equal(a, b)
