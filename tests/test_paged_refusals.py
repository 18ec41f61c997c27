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


def test_append_and_gather_of_overlapping_memory(lib):
    """Blocks of one row would write queries over rows that others still read."""
    c, H, ldq = _cache(), 2, 6 * 64
    x, rope, q = P16, P16 + 8192, P16 + 16384              # 4 rows of 1536 bytes, 4 of 256, 4 of 512

    def put(q_out, step=None, rope=rope):
        return _error(lib, lib.cgx_kv_paged_append_dev(C.byref(c), 0, C.byref(step or _step()), x, ldq, H, rope, 4, q_out))
    for bad in (x, x + 4 * 1536 - 16, x - 4 * 512 + 16, rope, rope + 1008):
        assert "overlap" in put(bad), bad - x
    assert "overlap" in put(x + 16, _step(rows=1))         # one row in place is fine, beside its place not
    assert "overlap" in put(q, _step(row_slot=q + 2032))
    assert "overlap" in put(q, _step(row_pos=q))
    for slots, k, v in ((x, q, q), (x, q, q + 1024), (q + 16, q, rope), (q, rope, q)):
        assert "overlap" in _error(lib, lib.cgx_kv_paged_gather_dev(C.byref(c), 0, slots, 4, k, v))


def test_attention_of_overlapping_memory(lib):
    c = _cache()
    Q, O, lse, ws = (P16 + k for k in (8192, 12288, 16384, 32768))     # 4 rows of 4 heads: 4096 bytes, 64 bytes

    def call(q=Q, o=O, lse=lse, **kw):
        step = _step(max_rows=1, **kw)
        assert not lib.cgx_attention_paged_ws(C.byref(c), C.byref(step), 4)
        return _error(lib, lib.cgx_attention_paged_dev(C.byref(c), 0, C.byref(step), q, 4, P16, P16 + 64, o, lse, ws, 0))
    for kw in (dict(o=Q + 16), dict(o=Q - 4080), dict(lse=Q), dict(lse=O + 4092), dict(o=Q, lse=Q), dict(o=P16 - 4080 + 64, q=O), dict(lse=P16 + 64),
               dict(table=O), dict(row_begin=O + 4092), dict(row_seq=lse + 60), dict(kv_len=lse)):
        assert "overlap" in call(**kw), kw
    # the workspace
    big = _step(max_rows=1, table_ld=256)
    need = lib.cgx_attention_paged_ws(C.byref(c), C.byref(big), 4)
    assert need
    for ws in (Q, O, O + 4080):
        e = _error(lib, lib.cgx_attention_paged_dev(C.byref(c), 0, C.byref(big), Q, 4, None, None, O, None, ws, need))
        assert "overlap" in e


def test_logprobs_of_overlapping_memory(lib):
    x, tok, lp, rank, ent, top, top_lp = (P16 + k for k in (0, 2048, 2112, 2176, 2240, 2304, 2368))   # 2 rows of 200, 3 alternatives

    def call(**kw):
        a = dict(x=x, tok=tok, lp=lp, rank=rank, ent=ent, top=top, top_lp=top_lp, ws=P16 + 4096, V=200) | kw
        V = a["V"]
        return _error(lib, lib.cgx_token_logprobs_dev(a["x"], V, 2, V, a["tok"], 3, a["lp"], a["rank"], a["ent"], a["top"],
                                                      a["top_lp"], a["ws"], 1 << 14))
    for kw in (dict(lp=x + 1596), dict(rank=tok + 4), dict(ent=lp), dict(top=ent + 4), dict(top_lp=top + 20),
               dict(V=9000, x=P16 + 16384, ws=P16 + 16384), dict(V=9000, x=P16 + 16384, lp=P16 + 4096)):
        assert "overlap" in call(**kw), kw


@pytest.mark.parametrize("layers,pages,heads,D", [
    (1 << 20, (1 << 27) - 1, 1 << 14, 32), (2**31 - 1, (1 << 27) - 1, 2**31 - 1, 256), (1 << 16, 1 << 26, 1 << 18, 64)])
def test_a_cache_whose_bytes_pass_64_bits(lib, layers, pages, heads, D):
    """Sizes that would wrap to a small allocation."""
    assert not lib.cgx_kv_paged_int4_new(layers, pages, 16, heads, D, D)
    assert "too large" in last_error(lib)
    lib.cgx_clear_error()
    c = _cache(num_layers=layers, num_pages=pages, n_heads=heads, head_dim=D, group_size=D)
    assert "too large" in _error(lib, lib.cgx_kv_paged_gather_dev(C.byref(c), 0, P16, 1, P16 + 4096, P16 + 8192))
