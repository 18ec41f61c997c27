"""CPU: calls of the serving steps that could only give wrong answers are refused before any device call."""
from __future__ import annotations

import ctypes as C

import pytest

from cogito_amd.capi import CgxKvPagedInt4, CgxPagedStep, last_error

_BUF = C.create_string_buffer(1 << 16)
P16 = (C.addressof(_BUF) + 15) & ~15                       # never read: the calls are refused first


def _cache(**kw):
    c = CgxKvPagedInt4(num_layers=1, num_pages=8, page_size=16, n_heads=2, head_dim=64, group_size=64)
    c.k_pages = c.v_pages = c.k_scales = c.v_scales = P16
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _step(**kw):
    s = CgxPagedStep(seqs=2, rows=4, max_rows=0, table_ld=4)
    for at, (name, _) in enumerate(CgxPagedStep._fields_[4:]):
        setattr(s, name, P16 + 4096 + 64 * at)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def _error(lib, rc):
    e = last_error(lib)
    lib.cgx_clear_error()
    assert rc == -1
    return e


@pytest.mark.parametrize("D", [64, 256])
def test_trees_of_more_rows_than_bits(lib, D):
    """A row's ancestor bits are 64: without tree_len a sequence's rows are its tree, and more of them cannot be told apart."""
    c = _cache(head_dim=D, group_size=D)

    def call(most, anc=P16, tree_len=None, rows=300):
        step = _step(rows=rows, max_rows=most, table_ld=256)
        if D > 128:
            rows = step.rows = min(rows, 100)              # few enough for a workspace there
        assert lib.cgx_attention_paged_ws(C.byref(c), C.byref(step), 4) > 0
        # without a workspace, which is refused last
        return _error(lib, lib.cgx_attention_paged_dev(C.byref(c), 0, C.byref(step), P16 + 8192, 4, anc, tree_len, P16 + 16384,
                                                       None, None, 0))
    assert "more than 64 rows" in call(65)
    assert "more than 64 rows" in call(300)
    # 64 of them, an unknown number, a window given, fewer rows in all, no tree
    for other in (call(64), call(0), call(300, tree_len=P16 + 128), call(300, rows=64), call(300, anc=None)):
        assert "workspace of" in other
