"""GPU: calls over the paged cache that other tests do not make: pages past 32
bits of byte offsets, a workspace with an earlier call's words, graphs that
share one, and the same call twice."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import paged_ref as R
from cogito_amd.capi import CgxPagedStep, DeviceArray, last_error

pytestmark = pytest.mark.gpu
TOL = 8e-6                      # per value, relative to sum_j p_j |v_j|: a score's roundings and the weights' two terms


def _up(lib, a, t=np.int32):
    return DeviceArray.from_numpy(lib, np.ascontiguousarray(a, t))


def _near(got, ref, rows):
    o, (O, _, A, F) = got[rows], (x if x is None else x[rows] for x in ref)
    assert np.all(np.abs(o - O) <= TOL * A + F + 1e-37)


def _call(b, o, ws, lse=None, q=None):
    lib = b.lib
    return lib.cgx_attention_paged_dev(C.byref(b.cache), b.layer, C.byref(b.step), (q or b.d["q"]).ptr, b.H, None, None,
                                       o.ptr, lse.ptr if lse else None, ws.ptr, ws.nbytes)


@pytest.mark.parametrize("H,Hk,D,gs", [(32, 8, 128, 128), (8, 8, 256, 256)])
def test_pages_past_32_bits(gpu, H, Hk, D, gs):
    """The same rows in a small cache and behind 4 GiB of pages: same values bit for bit. D 256 takes the other kernel."""
    rng = np.random.default_rng(D)
    P, T, kv = 256, 11, 700
    per_page = P * Hk * D // 2
    far = (1 << 32) // per_page + 5
    pages_of = R.pages_of(kv, P)
    got = []
    x = _up(gpu, rng.normal(size=(kv, (H + 2 * Hk) * D)), np.float32)
    qq = _up(gpu, rng.normal(size=(T, H, D)), np.float32)
    for first, pool in ((0, pages_of), (far, far + pages_of)):
        cache = gpu.cgx_kv_paged_int4_new(2, pool, P, Hk, D, gs)
        assert cache, last_error(gpu)
        table = first + np.arange(pages_of)[::-1]
        pos = np.arange(kv)
        slot = table[pos // P] * P + pos % P
        d = {k: _up(gpu, v) for k, v in dict(table=table, begin=[0, T], seq=[0] * T, kv=[kv], pos=pos, slot=slot).items()}
        st = CgxPagedStep(seqs=1, rows=kv, max_rows=0, table_ld=pages_of)
        st.row_slot, st.row_pos = d["slot"].ptr, d["pos"].ptr
        assert gpu.cgx_kv_paged_append_dev(cache, 1, C.byref(st), x.ptr, (H + 2 * Hk) * D, H, None, 0, None) == 0
        k, v = (DeviceArray(gpu, kv * Hk * D * 4) for _ in range(2))
        assert gpu.cgx_kv_paged_gather_dev(cache, 1, d["slot"].ptr, kv, k.ptr, v.ptr) == 0, last_error(gpu)
        st = CgxPagedStep(seqs=1, rows=T, max_rows=0, table_ld=pages_of)
        st.table, st.row_begin, st.row_seq, st.kv_len = (d[n].ptr for n in ("table", "begin", "seq", "kv"))
        n = gpu.cgx_attention_paged_ws(cache, C.byref(st), H)
        ws, o = DeviceArray(gpu, max(n, 16)), DeviceArray(gpu, T * H * D * 4)
        assert gpu.cgx_attention_paged_dev(cache, 1, C.byref(st), qq.ptr, H, None, None, o.ptr, None, ws.ptr, n) == 0
        assert gpu.cgx_synchronize() == 0, last_error(gpu)
        got.append([a.numpy(np.float32, (m,)) for a, m in ((k, kv * Hk * D), (v, kv * Hk * D), (o, T * H * D))])
        gpu.cgx_kv_paged_int4_free(cache)
    for a, b in zip(*got):
        assert np.abs(a).max() > 0
        np.testing.assert_array_equal(a, b)


def test_a_sequence_left_out_takes_nothing_from_an_earlier_call(gpu):
    """With max_rows below a sequence's rows its output stays, whatever the workspace holds of another call."""
    b = R.Batch(gpu, np.random.default_rng(21), [4000, 3000], [20, 1], 16, 8, 2, 128, 128, pad=1).bind()
    ref = b.reference()
    n = gpu.cgx_attention_paged_ws(C.byref(b.cache), C.byref(b.step), b.H)
    b.step.max_rows = 1
    n = max(n, gpu.cgx_attention_paged_ws(C.byref(b.cache), C.byref(b.step), b.H))
    ws = DeviceArray(gpu, n)
    for most in (0, 20, 1):
        b.step.max_rows = most
        o = _up(gpu, np.full((b.T, b.H, b.D), 7.0), np.float32)
        assert _call(b, o, ws) == 0 and gpu.cgx_synchronize() == 0, last_error(gpu)
        got = o.numpy(np.float32, (b.T, b.H, b.D))
        _near(got, ref, slice(0 if most != 1 else 20, 21))
        assert np.all(got[21:] == 7.0) and (most != 1 or np.all(got[:20] == 7.0))


def test_graphs_share_a_workspace(gpu):
    """Two captured calls and eager ones over one workspace, replayed in turn: each the same bits every time."""
    rng = np.random.default_rng(22)
    bs = [R.Batch(gpu, rng, [5000, 37, 900], [3, 2, 1], 16, 32, 8, 128, 128).bind(),
          R.Batch(gpu, rng, [2000, 64], [64, 5], 32, 12, 12, 64, 32).bind()]
    refs = [b.reference() for b in bs]
    ws = DeviceArray(gpu, max(gpu.cgx_attention_paged_ws(C.byref(b.cache), C.byref(b.step), b.H) for b in bs))
    outs = [(DeviceArray(gpu, b.T * b.H * b.D * 4), DeviceArray(gpu, b.T * b.H * 4)) for b in bs]
    first = []
    for b, (o, ls), ref in zip(bs, outs, refs):
        assert _call(b, o, ws, ls) == 0 and gpu.cgx_synchronize() == 0, last_error(gpu)
        first.append((o.numpy(np.uint32, (b.T * b.H * b.D,)), ls.numpy(np.uint32, (b.T * b.H,))))
        _near(o.numpy(np.float32, (b.T, b.H, b.D)), ref, slice(0, b.T))
        assert np.all(np.abs(ls.numpy(np.float32, (b.T, b.H)) - ref[1]) <= TOL * (1 + np.abs(ref[1])))
    graphs = []
    for b, (o, ls) in zip(bs, outs):
        assert gpu.cgx_graph_begin() == 0
        rc = _call(b, o, ws, ls)
        graphs.append(gpu.cgx_graph_end())
        assert rc == 0 and graphs[-1], last_error(gpu)
    for turn in range(4):
        for i in ((0, 1), (1, 0), (0, 0), (1, 1))[turn]:
            b, (o, ls) = bs[i], outs[i]
            o.upload(np.full(b.T * b.H * b.D, 7.0, np.float32))
            assert gpu.cgx_graph_launch(graphs[i]) == 0
            other = bs[1 - i]                              # an eager call behind it, on the same workspace
            assert _call(other, outs[1 - i][0], ws, outs[1 - i][1]) == 0 and gpu.cgx_synchronize() == 0, last_error(gpu)
            for j, bj in enumerate(bs):
                np.testing.assert_array_equal(outs[j][0].numpy(np.uint32, (bj.T * bj.H * bj.D,)), first[j][0])
                np.testing.assert_array_equal(outs[j][1].numpy(np.uint32, (bj.T * bj.H,)), first[j][1])
    for g in graphs:
        assert gpu.cgx_graph_free(g) == 0


@pytest.mark.parametrize("seqs", [64, 65, 300])
def test_many_sequences_of_mixed_rows(gpu, seqs):
    """More sequences than lanes, with none, one and many rows, some without keys, cut and whole."""
    rng = np.random.default_rng(seqs)
    kv = [int(k) for k in rng.integers(0, 90, seqs)]
    rows = [int(min(k, r)) for k, r in zip(kv, rng.integers(0, 4, seqs))]
    kv[seqs // 2], rows[seqs // 2] = 2500, 40
    kv[-1], rows[-1] = 1300, 2
    b = R.Batch(gpu, rng, kv, rows, 16, 4, 2, 64, 64, pad=2).bind()
    ref = b.reference()
    for most in (0, 40):
        o, _ = b.attend(max_rows=most)
        n = int(b.begin[-1])
        _near(o, ref, slice(0, n))
        assert np.all(o[n:] == 7.0)


def test_logprob_graphs_share_a_workspace(gpu):
    """Rows of several segments: a captured call replayed behind eager calls of another shape, bit for bit."""
    rng = np.random.default_rng(23)
    sets = []
    for rows, V, n in ((5, 32000, 20), (40, 9001, 5)):
        x = rng.normal(size=(rows, V)).astype(np.float32) * 3
        sets.append(dict(rows=rows, V=V, n=n, x=_up(gpu, x, np.float32), tok=_up(gpu, rng.integers(0, V, rows)),
                         out=[DeviceArray(gpu, rows * 4) for _ in range(3)] +
                             [DeviceArray(gpu, rows * n * 4) for _ in range(2)]))
    ws = DeviceArray(gpu, max(gpu.cgx_token_logprobs_ws(s["rows"], s["V"], s["n"]) for s in sets))

    def call(s):
        return gpu.cgx_token_logprobs_dev(s["x"].ptr, s["V"], s["rows"], s["V"], s["tok"].ptr, s["n"],
                                          *(a.ptr for a in s["out"]), ws.ptr, ws.nbytes)

    def bits(s):
        return [a.numpy(np.uint32, (a.nbytes // 4,)) for a in s["out"]]
    first = []
    for s in sets:
        assert call(s) == 0 and gpu.cgx_synchronize() == 0, last_error(gpu)
        first.append(bits(s))
    assert gpu.cgx_graph_begin() == 0
    rc = call(sets[0])
    g = gpu.cgx_graph_end()
    assert rc == 0 and g, last_error(gpu)
    for _ in range(4):
        for a in sets[0]["out"]:
            a.upload(np.zeros(a.nbytes // 4, np.uint32))
        assert call(sets[1]) == 0 and gpu.cgx_graph_launch(g) == 0 and gpu.cgx_synchronize() == 0, last_error(gpu)
        for s, f in zip(sets, first):
            for a, b in zip(bits(s), f):
                np.testing.assert_array_equal(a, b)
    assert gpu.cgx_graph_free(g) == 0


@pytest.mark.parametrize("H,Hk,D,gs", [(4, 2, 256, 256), (2, 2, 192, 24), (3, 1, 64, 16)])
@pytest.mark.parametrize("tree", [False, True])
def test_rows_of_other_heads_over_long_keys(gpu, H, Hk, D, gs, tree):
    """Head sizes and scale groups off the matrix cores: keys cut over blocks, pieces without keys, rows without."""
    rng = np.random.default_rng(D + gs)
    b = R.Batch(gpu, rng, [3000, 5, 0, 257], [3, 2, 1, 9], 16, H, Hk, D, gs, pad=2).bind()
    anc = [int(x) for x in rng.integers(0, 1 << 9, b.T)] if tree else None
    ref, got = b.reference(anc=anc), b.attend(anc=anc)
    n = int(b.begin[-1])
    _near(got[0], ref, slice(0, n))
    fin = np.isfinite(ref[1][:n])
    np.testing.assert_array_equal(got[1][:n][~fin], ref[1][:n][~fin])
    g, e = got[1][:n][fin], ref[1][:n][fin]
    assert np.all(np.abs(g - e) <= TOL * (1 + np.abs(e)))
    assert np.all(got[0][n:] == 7.0) and np.all(got[1][n:] == 7.0)


def test_the_most_sequences(gpu):
    """4096 sequences, 64 a lane of the search, most of a key or two and some without rows or keys."""
    rng = np.random.default_rng(24)
    kv = [int(k) for k in rng.integers(0, 4, 4096)]
    rows = [int(min(k, r)) for k, r in zip(kv, rng.integers(0, 3, 4096))]
    for i, (k, n) in {0: (900, 1), 777: (40, 33), 2048: (2000, 3), 4095: (70, 20)}.items():
        kv[i], rows[i] = k, n
    b = R.Batch(gpu, rng, kv, rows, 16, 2, 1, 32, 32, pad=3).bind()
    ref, (o, _) = b.reference(), b.attend()
    n = int(b.begin[-1])
    _near(o, ref, slice(0, n))
    assert np.all(o[n:] == 7.0)
