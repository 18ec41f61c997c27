"""CPU: the paged cache's and the log probabilities' entry points refuse bad
arguments before any device call."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from cogito_amd.capi import CgxKvPagedInt4, CgxPagedStep, last_error

_BUF = C.create_string_buffer(1 << 16)
P16 = (C.addressof(_BUF) + 15) & ~15


def _cache(**kw):
    c = CgxKvPagedInt4(num_layers=2, num_pages=8, page_size=16, n_heads=2, head_dim=64, group_size=64)
    c.k_pages, c.v_pages, c.k_scales, c.v_scales = P16, P16 + 1024, P16 + 2048, P16 + 4096
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _step(**kw):
    s = CgxPagedStep(seqs=2, rows=4, max_rows=0, table_ld=4)
    at = P16 + 8192
    for name, _ in CgxPagedStep._fields_[4:]:
        if name != "table_old":
            setattr(s, name, at)
        at += 256
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def _refused(lib, rc, word):
    assert rc == -1
    assert word in last_error(lib), last_error(lib)
    lib.cgx_clear_error()


def test_struct_sizes():
    assert C.sizeof(CgxKvPagedInt4) == 56 and C.sizeof(CgxPagedStep) == 104


@pytest.mark.parametrize("bad", [dict(page_size=8), dict(page_size=48), dict(page_size=8192), dict(head_dim=48),
                                 dict(head_dim=288), dict(group_size=3), dict(group_size=24), dict(group_size=0),
                                 dict(num_pages=0), dict(n_heads=0), dict(num_layers=0),
                                 dict(num_pages=2**27, page_size=16)])
def test_cache_shapes(lib, bad):
    c = _cache(**bad)
    args = [getattr(c, k) for k in ("num_layers", "num_pages", "page_size", "n_heads", "head_dim", "group_size")]
    assert not lib.cgx_kv_paged_int4_new(*args)
    assert "cgx_kv_paged_int4_new" in last_error(lib)
    lib.cgx_clear_error()
    s = _step()
    _refused(lib, lib.cgx_attention_paged_dev(C.byref(c), 0, C.byref(s), P16, 2, None, None, P16, None, P16, 1 << 30),
             "page_size a power of two")
    _refused(lib, lib.cgx_kv_paged_append_dev(C.byref(c), 0, C.byref(s), P16, 4096, 2, None, 0, None),
             "page_size a power of two")
    _refused(lib, lib.cgx_kv_paged_gather_dev(C.byref(c), 0, P16, 1, P16, P16), "page_size a power of two")


@pytest.mark.parametrize("bad,word", [
    (dict(page=8), "power of two"), (dict(page=24), "power of two"), (dict(pages=0), "pages of"),
    (dict(step=dict(seqs=0)), "a step of"), (dict(step=dict(seqs=4097)), "a step of"),
    (dict(step=dict(rows=-1)), "a step of"), (dict(step=dict(max_rows=-1)), "a step of"),
    (dict(step=dict(table_ld=0)), "a step of"), (dict(step=dict(table_ld=2**28)), "a step of"),
    (dict(step=dict(kv_old=None)), "required"), (dict(step=dict(table=None)), "required"),
    (dict(step=dict(row_slot=None)), "required"), (dict(step=dict(status=None)), "required"),
    (dict(free=None), "required"), (dict(count=None), "required"), (dict(left=None), "required"),
    (dict(alias=("kv_len", "kv_old")), "overlaps an input"), (dict(alias=("kv_len", "rows_new")), "overlaps an input"),
    (dict(alias=("row_begin", "kv_keep")), "overlaps an input"), (dict(alias=("row_pos", "row_slot")), "two outputs"),
    (dict(left="count"), "overlaps an input"), (dict(partial=True), "overlaps an input")])
def test_plan_arguments(lib, bad, word):
    s = _step(**bad.get("step", {}))
    free, count = bad.get("free", P16), bad.get("count", P16 + 512)
    left = bad.get("left", P16 + 768)
    left = count if left == "count" else left
    if "alias" in bad:
        setattr(s, bad["alias"][0], getattr(s, bad["alias"][1]))
    if bad.get("partial"):
        s.table_old = s.table + 4                          # neither apart nor the same
    _refused(lib, lib.cgx_paged_plan_dev(C.byref(s), bad.get("page", 16), bad.get("pages", 8), free, count, left), word)
    _refused(lib, lib.cgx_paged_plan_dev(None, 16, 8, P16, P16 + 512, P16 + 768), "a step of")


def test_append_arguments(lib):
    c, s = _cache(), _step()
    ldq = (4 + 4) * 64

    def call(cache=c, layer=0, step=s, qkv=P16, ldq=ldq, H=4, rope=P16, rope_rows=4, q=P16):
        return lib.cgx_kv_paged_append_dev(C.byref(cache) if cache else None, layer, C.byref(step), qkv, ldq, H, rope,
                                           rope_rows, q)
    _refused(lib, call(cache=None), "no cache")
    _refused(lib, call(cache=_cache(v_scales=None)), "no cache")
    _refused(lib, call(cache=_cache(k_pages=P16 + 4)), "16-byte aligned")
    _refused(lib, call(layer=2), "layer 2 of 2")
    _refused(lib, call(layer=-1), "layer -1 of 2")
    _refused(lib, call(qkv=None), "qkv rows")
    _refused(lib, call(ldq=ldq - 4), "qkv rows")
    _refused(lib, call(H=-1), "qkv rows")
    _refused(lib, call(rope_rows=0), "qkv rows")
    _refused(lib, call(step=_step(row_slot=None)), "row_slot")
    _refused(lib, call(step=_step(row_pos=None)), "row_pos")
    _refused(lib, call(ldq=ldq + 2), "multiple of 4")
    _refused(lib, call(qkv=P16 + 4), "16-byte aligned")
    _refused(lib, call(q=P16 + 8), "16-byte aligned")
    _refused(lib, lib.cgx_kv_paged_gather_dev(C.byref(c), 0, None, 1, P16, P16), "slots")
    _refused(lib, lib.cgx_kv_paged_gather_dev(C.byref(c), 0, P16, -1, P16, P16), "slots")
    _refused(lib, lib.cgx_kv_paged_gather_dev(C.byref(c), 0, P16, 1, P16, P16 + 4), "slots")


def test_attention_arguments(lib):
    c, s = _cache(), _step()

    def call(cache=c, layer=0, step=s, q=P16, H=4, anc=None, tree=None, o=P16, lse=None, ws=P16, n=1 << 30):
        return lib.cgx_attention_paged_dev(C.byref(cache), layer, C.byref(step), q, H, anc, tree, o, lse, ws, n)
    _refused(lib, call(layer=5), "layer 5")
    _refused(lib, call(step=_step(seqs=0)), "a step of")
    _refused(lib, call(H=3), "3 query heads over 2")
    _refused(lib, call(H=0), "0 query heads")
    _refused(lib, call(q=None), "Q, O")
    _refused(lib, call(o=None), "Q, O")
    _refused(lib, call(q=P16 + 4), "16-byte aligned")
    for k in ("table", "row_begin", "row_seq", "kv_len"):
        _refused(lib, call(step=_step(**{k: None})), "required")
    _refused(lib, call(tree=P16), "without ancestor bits")
    need = lib.cgx_attention_paged_ws(C.byref(c), C.byref(s), 4)
    if need:
        _refused(lib, call(n=need - 1), "workspace")
        _refused(lib, call(ws=None), "workspace")
        _refused(lib, call(ws=P16 + 4), "workspace")
    assert lib.cgx_attention_paged_ws(C.byref(c), C.byref(s), 3) == 0
    assert "query heads" in last_error(lib)
    lib.cgx_clear_error()


def test_logprob_arguments(lib):
    def call(x=P16, ld=100, rows=2, V=100, tok=P16, n=3, lp=P16, rank=P16, ent=P16, top=P16, top_lp=P16, ws=P16,
             nb=1 << 30):
        return lib.cgx_token_logprobs_dev(x, ld, rows, V, tok, n, lp, rank, ent, top, top_lp, ws, nb)
    _refused(lib, call(x=None), "rows of V")
    _refused(lib, call(ld=99), "rows of V")
    _refused(lib, call(rows=-1), "rows of V")
    _refused(lib, call(V=0), "rows of V")
    _refused(lib, call(n=33), "0..32")
    _refused(lib, call(n=-1), "0..32")
    _refused(lib, call(tok=None), "need the tokens")
    _refused(lib, call(tok=None, lp=None), "need the tokens")
    _refused(lib, call(top=None), "n_top > 0")
    _refused(lib, call(top_lp=None), "n_top > 0")
    _refused(lib, call(n=0), "n_top > 0")
    need = lib.cgx_token_logprobs_ws(2, 100, 3)
    if need:
        _refused(lib, call(nb=need - 1), "workspace")
        _refused(lib, call(ws=P16 + 8), "workspace")
        _refused(lib, call(ws=None), "workspace")
    assert lib.cgx_token_logprobs_ws(2, 100, 33) == 0
    lib.cgx_clear_error()


def test_the_reference_plan_keeps_every_page_once():
    """The reference plan itself: pages are conserved, and a refused step leaves everything."""
    rng = np.random.default_rng(0)
    for _ in range(50):
        B, P, ld = int(rng.integers(1, 9)), 16, 6
        old = rng.integers(0, 60, B)
        held = [R.pages_of(n, P) for n in old]
        pages = sum(held) + 12
        order = rng.permutation(pages)
        table, at = np.full((B, ld), -1), 0
        for b in range(B):
            table[b, :held[b]] = order[at:at + held[b]]
            at += held[b]
        free = np.full(pages, -1)
        free[:12] = order[at:]
        keep, new = old - np.minimum(old, rng.integers(0, 30, B)), rng.integers(0, 30, B)
        bits, out = R.plan(old, keep, new, table, P, free, 12, 400, ld, pages)
        if bits:
            assert bits == 8 and out["left"] == 12
            continue
        live = np.concatenate([out["table"][b, :R.pages_of(keep[b] + new[b], P)] for b in range(B)])
        assert sorted(np.concatenate([live, out["free"][:out["left"]]]).tolist()) == list(range(pages))


def test_sizes_past_a_launch_are_refused(lib):
    """Row counts, positions and vocabularies whose grids or indices would not fit."""
    c, s = _cache(), _step()
    big = _step(rows=2**23)
    _refused(lib, lib.cgx_paged_plan_dev(C.byref(big), 16, 8, P16, P16 + 512, P16 + 768), "a step of")
    _refused(lib, lib.cgx_kv_paged_append_dev(C.byref(c), 0, C.byref(big), P16, 512, 4, None, 0, None), "a step of")
    _refused(lib, lib.cgx_kv_paged_gather_dev(C.byref(c), 0, P16, 2**23, P16, P16), "slots")
    long = _step(table_ld=2**26 + 1)                       # 16 positions an entry
    _refused(lib, lib.cgx_attention_paged_dev(C.byref(c), 0, C.byref(long), P16, 2, None, None, P16, None, P16, 1 << 40),
             "2^30 positions")
    _refused(lib, lib.cgx_paged_plan_dev(C.byref(long), 16, 8, P16, P16 + 512, P16 + 768), "2^30 positions")

    def attend(cache, step, H):
        return lib.cgx_attention_paged_dev(C.byref(cache), 0, C.byref(step), P16, H, None, None, P16, None, P16, 1 << 40)
    _refused(lib, attend(c, s, 65536), "65536 query heads")
    _refused(lib, attend(c, _step(rows=2**22), 1024), "too many for one call")            # rows times heads
    _refused(lib, attend(_cache(n_heads=32768), _step(seqs=4096, rows=4096), 32768), "too many for one call")
    assert lib.cgx_attention_paged_ws(C.byref(c), C.byref(_step(rows=2**22)), 1024) == 0
    assert "too many" in last_error(lib)

    def logprobs(rows, V):
        return lib.cgx_token_logprobs_dev(P16, 1 << 31, rows, V, P16, 0, P16, P16, P16, None, None, P16, 1 << 40)
    _refused(lib, logprobs(2**23, 10), "fewer than 2^23 rows")
    _refused(lib, logprobs(1, 2**30 + 1), "V at most 2^30")
    assert lib.cgx_token_logprobs_ws(1, 2**30 + 1, 0) == 0
    lib.cgx_clear_error()
