"""GPU: a step that only gives pages back: no row arrays."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from cogito_amd.capi import CgxPagedStep, DeviceArray, last_error

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows_at", [None, 8])
def test_a_plan_without_rows(gpu, rows_at):
    """Row pointers of a step of no rows may be anything: none, or in the middle of another array."""
    up = lambda a: DeviceArray.from_numpy(gpu, np.asarray(a, np.int32))   # noqa: E731
    P, ld, pages = 16, 3, 9
    old, keep, new = [40, 16, 0, 33], [0, 16, 0, 20], [0, 0, 0, 0]
    table = [[4, 0, 7], [2, -5, -5], [-5, -5, -5], [1, 8, 3]]
    free = [5, 6, -1, -1, -1, -1, -1, -1, -1]
    bits, exp = R.plan(old, keep, new, table, P, free, 2, 0, ld, pages)
    assert bits == 0 and exp["left"] == 6
    d = dict(old=up(old), keep=up(keep), new=up(new), table=up(table), begin=up([-9] * 5), kv=up([-9] * 4), status=up([-9] * 4),
             free=up(free), count=up([2]), left=up([-9]))
    st = CgxPagedStep(seqs=4, rows=0, max_rows=0, table_ld=ld)
    st.kv_old, st.kv_keep, st.rows_new, st.table = (d[k].ptr for k in ("old", "keep", "new", "table"))
    st.row_begin, st.kv_len, st.status = (d[k].ptr for k in ("begin", "kv", "status"))
    if rows_at:
        st.row_seq = st.row_pos = st.row_slot = d["status"].ptr + rows_at
    assert gpu.cgx_paged_plan_dev(C.byref(st), P, pages, d["free"].ptr, d["count"].ptr, d["left"].ptr) == 0, last_error(gpu)
    assert gpu.cgx_synchronize() == 0, last_error(gpu)
    get = lambda k, n: d[k].numpy(np.int32, (n,)).tolist()             # noqa: E731
    assert get("begin", 5) == [0] * 5 and get("kv", 4) == exp["kv"].tolist() and get("status", 4) == exp["status"]
    assert get("left", 1) == [6] and get("free", pages) == exp["free"].tolist()
    assert get("table", 4 * ld) == np.ravel(table).tolist()            # in place: nothing taken
