"""GPU: a slot that two rows of an append are given."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from cogito_amd.capi import CgxPagedStep, DeviceArray, last_error

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Hk,D,gs", [(8, 128, 128), (3, 96, 32), (2, 64, 2)])
def test_a_slot_given_twice_touches_no_other(gpu, Hk, D, gs):
    """Its bytes and scales are one row's or the other's each, of one row where both are the same; every other position
    is as without the second row."""
    rng = np.random.default_rng(D)
    T, P, pages = 12, 16, 3
    x = rng.normal(size=(T, 2 * Hk * D)).astype(np.float32)
    x[9] = x[4]
    slot = rng.permutation(pages * P)[:T]
    slot[7], slot[9] = slot[2], slot[4]                    # rows 2 and 7 differ, 4 and 9 are the same
    pool = R.Pool(1, pages, P, Hk, D, gs)
    cache = pool.upload(gpu)
    dx, ds = DeviceArray.from_numpy(gpu, x), DeviceArray.from_numpy(gpu, slot.astype(np.int32))
    st = CgxPagedStep(seqs=1, rows=T, max_rows=0, table_ld=1)
    st.row_slot = ds.ptr
    assert gpu.cgx_kv_paged_append_dev(C.byref(cache), 0, C.byref(st), dx.ptr, x.shape[1], 0, None, 0, None) == 0
    assert gpu.cgx_synchronize() == 0, last_error(gpu)
    got = pool.download()
    want = []
    kc, ks = R.quantise(x[:, :Hk * D].reshape(T, Hk, D), gs)
    vc, vs = R.quantise(x[:, Hk * D:].reshape(T, Hk, D), gs)
    for second in (2, 7):
        for t in range(T):
            if t not in (2, 7) or t == second:
                pool.put(0, int(slot[t]), kc[t], ks[t], vc[t], vs[t])
        want.append([a.copy() for a in (pool.k, pool.v, pool.ks, pool.vs)])
    for g, a, b in zip(got, *want):
        same = lambda p, q: (p == q) | ((p != p) & (q != q))   # noqa: E731  (positions nobody wrote hold NaN)
        assert np.all(same(g, a) | same(g, b))
        assert np.any(~same(a, b))
