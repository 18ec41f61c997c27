"""CPU: workspaces of the serving steps.  A program sizes one for the largest
call that it makes and passes it to every smaller one, so a size never falls
as a call grows."""
from __future__ import annotations

import ctypes as C

import pytest

from cogito_amd.capi import CgxKvPagedInt4, CgxPagedStep, last_error

_BUF = C.create_string_buffer(256)
P16 = (C.addressof(_BUF) + 15) & ~15                       # never read: the calls are refused first

# either side of every bound on the rows that the choice of segments has
ROWS = sorted({r + d for r in (1, 2, 8, 9, 16, 32, 63, 64, 128, 255, 256, 342, 512, 1000, 1024, 4096)
               for d in (-1, 0, 1)} - {0})


@pytest.mark.parametrize("n_top", [0, 1, 20, 32])
def test_logprob_workspaces_grow_with_the_call(lib, n_top):
    before = [0] * len(ROWS)
    for V in (1, 4096, 4097, 8192, 8193, 9000, 12289, 32000, 50257, 128256, 262145, 600000, 1 << 30):
        need = [lib.cgx_token_logprobs_ws(r, V, n_top) for r in ROWS]
        assert need == sorted(need), V                                 # rows
        assert all(a <= b for a, b in zip(before, need)), V            # vocabulary
        if n_top:
            assert all(lib.cgx_token_logprobs_ws(r, V, n_top - 1) <= n for r, n in zip(ROWS, need))
        before = need
    assert lib.cgx_token_logprobs_ws(0, 32000, n_top) == 0


def _sizes(lib, shape, table_lds, steps, H):
    cache = CgxKvPagedInt4(num_layers=1, num_pages=64, page_size=16, **shape)
    out = []
    lib.cgx_clear_error()
    for ld in table_lds:
        for kw in steps:
            s = CgxPagedStep(table_ld=ld, **kw)
            out.append(lib.cgx_attention_paged_ws(C.byref(cache), C.byref(s), H))
            assert last_error(lib) == ""
    return out


# the two kernels: heads of 128 and less on the matrix cores, the others
SHAPES = [(dict(n_heads=8, head_dim=128, group_size=128), 32), (dict(n_heads=12, head_dim=64, group_size=32), 12),
          (dict(n_heads=2, head_dim=96, group_size=32), 16), (dict(n_heads=1, head_dim=32, group_size=32), 1),
          (dict(n_heads=8, head_dim=256, group_size=256), 8), (dict(n_heads=2, head_dim=64, group_size=16), 2),
          (dict(n_heads=4, head_dim=192, group_size=24), 300)]


@pytest.mark.parametrize("shape,H", SHAPES)
def test_attention_workspaces_grow_with_the_step(lib, shape, H):
    lds = (1, 16, 17, 24, 36, 38, 40, 64, 65, 256, 4096, 1 << 20)
    for seqs in (1, 2, 3, 64, 4096):
        for most in (0, 1, 2, 5, 40, 4000):
            # rows
            for ld in lds:
                need = _sizes(lib, shape, [ld], [dict(seqs=seqs, rows=r, max_rows=most) for r in ROWS], H)
                assert need == sorted(need), (seqs, most, ld)
            # positions a sequence
            need = _sizes(lib, shape, lds, [dict(seqs=seqs, rows=65, max_rows=most)], H)
            assert need == sorted(need), (seqs, most)
    for rows in ROWS:
        # sequences, and rows of one of them (0: any number)
        for most in (0, 1, 4, 33):
            need = _sizes(lib, shape, [300], [dict(seqs=s, rows=rows, max_rows=most) for s in (1, 2, 3, 5, 64, 65, 4096)], H)
            assert need == sorted(need), (rows, most)
        for seqs in (1, 2, 64):
            need = _sizes(lib, shape, [300], [dict(seqs=seqs, rows=rows, max_rows=m) for m in (1, 2, 4, 5, 8, 9, 17, 33, 400, 0)], H)
            assert need == sorted(need), (rows, seqs)


@pytest.mark.parametrize("shape,H,kw", [
    (dict(n_heads=2, head_dim=64, group_size=64), 4, dict(seqs=2, rows=4, max_rows=1)),        # a split launch
    (dict(n_heads=2, head_dim=64, group_size=64), 64, dict(seqs=1, rows=4)),                   # tiles of 64 rows
    (dict(n_heads=2, head_dim=256, group_size=256), 4, dict(seqs=2, rows=4))])                 # off the matrix cores
def test_attention_refuses_other_workspaces(lib, shape, H, kw):
    c = CgxKvPagedInt4(num_layers=1, num_pages=64, page_size=16, **shape)
    c.k_pages, c.v_pages, c.k_scales, c.v_scales = P16, P16, P16, P16
    s = CgxPagedStep(table_ld=256, **kw)
    s.table, s.row_begin, s.row_seq, s.kv_len = P16, P16, P16, P16
    need = lib.cgx_attention_paged_ws(C.byref(c), C.byref(s), H)
    assert need > 0, last_error(lib)
    for ws, n in ((P16, need - 1), (P16, 0), (None, need), (P16 + 4, need), (None, 0)):
        assert lib.cgx_attention_paged_dev(C.byref(c), 0, C.byref(s), P16, H, None, None, P16, None, ws, n) == -1
        assert "workspace of" in last_error(lib)
        lib.cgx_clear_error()


@pytest.mark.parametrize("rows,V,n_top", [(2, 9000, 3), (5, 32000, 0), (4096, 12000, 20)])
def test_logprobs_refuse_other_workspaces(lib, rows, V, n_top):
    top = P16 if n_top else None
    need = lib.cgx_token_logprobs_ws(rows, V, n_top)
    assert need > 0
    for ws, n in ((P16, need - 1), (P16, 0), (None, need), (P16 + 8, need), (None, 0)):
        assert lib.cgx_token_logprobs_dev(P16, V, rows, V, P16, n_top, P16, P16, P16, top, top, ws, n) == -1
        assert "workspace of" in last_error(lib)
        lib.cgx_clear_error()
