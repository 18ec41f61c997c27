"""GPU: the paged INT4 cache's tables, append, read-back and attention against
plain numpy, and a step captured into a graph.

Tolerance of the attention, per output value: 8e-6 times A = sum_j p_j |v_j|.
A score is a sum of D products in fp32 and its exponent's argument, |s| up to
about 20, is rounded three times (20 * 3 * 2^-24 = 3.6e-6 relative in p);
weights are carried as hi + lo fp16 (2^-22 = 2.4e-7) and added over the keys in
fp32, whose roundings at 4096 keys add up like sqrt(4096) * 2^-24 = 3.8e-6.
Beside it stands what a fixed-point pair of fp16 terms cannot hold: a row's
weights w_j = p_j s_j (s_j the V scale) are brought below 2^15 by one power of
two, so each is off by at most half the spacing of fp16's subnormals, 2^-25,
in units of max w 2^-14, and a code is at most 8: over N keys N 2^-36 max w.
That is seen where the keys of large weight have the code 0 in a dimension.
lse: the same score error, absolute, 8e-6 * (1 + |lse|)."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import oracle_lib
import paged_ref as R
from cogito_amd.capi import CgxPagedStep, DeviceArray, last_error

pytestmark = pytest.mark.gpu
TOL = 8e-6


def _dev(lib, a, t=np.int32):
    return DeviceArray.from_numpy(lib, np.asarray(a, t))


# ------------------------------------------------------------------ tables

class Plan:
    def __init__(self, lib, old, keep, new, table, P, free, count, rows, num_pages, in_place, max_rows=0):
        self.lib, B, ld = lib, len(old), table.shape[1]
        self.d = dict(old=_dev(lib, old), new=_dev(lib, new), told=_dev(lib, table), free=_dev(lib, free),
                      count=_dev(lib, [count]), left=_dev(lib, [-9]))
        self.shape = dict(begin=(B + 1,), seq=(rows,), pos=(rows,), slot=(rows,), kv=(B,), status=(4,))
        for k, s in self.shape.items():
            self.d[k] = _dev(lib, np.full(max(1, s[0]) + 4, -9))       # guard words behind
        self.d["keep"] = _dev(lib, keep) if keep is not None else None
        self.d["table"] = self.d["told"] if in_place else _dev(lib, np.full((B, ld), -9))
        st = CgxPagedStep(seqs=B, rows=rows, max_rows=max_rows, table_ld=ld)
        st.kv_old, st.rows_new, st.table = (self.d[k].ptr for k in ("old", "new", "table"))
        st.kv_keep = self.d["keep"].ptr if keep is not None else None
        st.table_old = None if in_place else self.d["told"].ptr
        st.row_begin, st.row_seq, st.row_pos, st.row_slot, st.kv_len, st.status = (
            self.d[k].ptr for k in ("begin", "seq", "pos", "slot", "kv", "status"))
        self.step, self.args = st, (P, num_pages, self.d["free"].ptr, self.d["count"].ptr, self.d["left"].ptr)
        self.B, self.ld, self.num_pages = B, ld, num_pages

    def run(self):
        assert self.lib.cgx_paged_plan_dev(C.byref(self.step), *self.args) == 0, last_error(self.lib)
        assert self.lib.cgx_synchronize() == 0, last_error(self.lib)
        out = {}
        for k, s in self.shape.items():
            a = self.d[k].numpy(np.int32, (max(1, s[0]) + 4,))
            assert np.all(a[s[0]:] == -9), k
            out[k] = a[:s[0]]
        out["left"] = int(self.d["left"].numpy(np.int32, (1,))[0])
        out["free"] = self.d["free"].numpy(np.int32, (self.num_pages,))
        out["table"] = self.d["table"].numpy(np.int32, (self.B, self.ld))
        return out


def _state(rng, B, ctx, P, ld, spare):
    old = rng.integers(0, ctx + 1, B)
    held = [R.pages_of(n, P) for n in old]
    pages = sum(held) + spare
    order = rng.permutation(pages)
    table = np.full((B, ld), -5, np.int64)                 # entries nobody reads
    at = 0
    for b in range(B):
        table[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
    free = np.full(pages, -1, np.int64)
    free[:spare] = order[at:]
    return old, table, free, pages


@pytest.mark.parametrize("B,ctx,most,P,in_place", [
    (1, 0, 1, 16, False), (1, 40, 1, 16, True), (3, 17, 40, 16, False), (64, 300, 5, 16, True),
    (64, 300, 5, 16, False), (65, 200, 97, 64, False), (257, 90, 3, 32, True), (1000, 64, 9, 16, False),
    (4096, 33, 2, 16, True), (7, 9000, 1, 4096, False)])
@pytest.mark.parametrize("rollback", [False, True])
def test_plan(gpu, B, ctx, most, P, in_place, rollback):
    rng = np.random.default_rng(B + ctx + most + rollback)
    ld = R.pages_of(ctx + most, P) + 2
    old, table, free, pages = _state(rng, B, ctx, P, ld, spare=B * (R.pages_of(most, P) + 1) + 3)
    count = int(np.sum(free >= 0))
    new = rng.integers(0, most + 1, B)
    keep = None
    if rollback:
        keep = np.maximum(0, old - rng.integers(0, 2 * P, B))
        ended = rng.random(B) < 0.2                         # ended requests: nothing kept or added
        keep[ended], new[ended] = 0, 0
    rows = int(new.sum()) + 5
    bits, exp = R.plan(old, keep if rollback else old, new, table, P, free, count, rows, ld, pages)
    assert bits == 0
    p = Plan(gpu, old, keep, new, table, P, free, count, rows, pages, in_place)
    for rep in range(1 if in_place else 2):                # another table: the same step again
        got = p.run()
        for k in ("begin", "seq", "pos", "slot", "kv", "left", "free", "status"):
            np.testing.assert_array_equal(got[k], exp[k], err_msg=k)
        for b in range(B):
            n = R.pages_of(exp["kv"][b], P)
            np.testing.assert_array_equal(got["table"][b, :n], exp["table"][b, :n])
            past = got["table"][b, n:]
            assert np.array_equal(past, table[b, n:]) if in_place else np.all(past == -1)
    # every page is held once: in a table or on the stack
    live = [exp["table"][b, :R.pages_of(exp["kv"][b], P)] for b in range(B)]
    assert sorted(np.concatenate(live + [exp["free"][:exp["left"]]])) == list(range(pages))


@pytest.mark.parametrize("what,bits", [
    ("keep", 1), ("negative", 1), ("wide", 2), ("rows", 4), ("max_rows", 4), ("pages", 8), ("count", 16),
    ("stack", 16), ("huge", 2)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_refuses_the_whole_step(gpu, what, bits, in_place):
    rng = np.random.default_rng(5)
    B, P, ld = 6, 16, 5
    old, table, free, pages = _state(rng, B, 50, P, ld, spare=20)
    count, keep, new, rows, max_rows = 20, np.array(old), np.full(B, 3), 40, 0
    if what == "keep":
        keep[2] = old[2] + 1
    elif what == "negative":
        new[1] = -1
    elif what == "wide":
        new[4] = ld * P + 1 - keep[4]
        rows = 200
    elif what == "huge":
        new[4] = 2**31 - 1
        rows = 200
    elif what == "rows":
        rows = 17
    elif what == "max_rows":
        max_rows = 2
    elif what == "pages":
        count, new = 1, np.full(B, 17)
        rows = 200
    elif what == "count":
        count = pages + 1
    else:
        keep, new = np.zeros(B, int), np.zeros(B, int)     # gives more back than the stack holds
        count = pages - 1
    exp_bits, exp = R.plan(old, keep, new, table, P, free, count, rows, ld, pages, max_rows)
    assert exp_bits == bits
    p = Plan(gpu, old, keep, new, table, P, free, count, rows, pages, in_place, max_rows)
    got = p.run()
    for k in ("begin", "seq", "pos", "slot", "kv", "left", "free", "status", "table"):
        np.testing.assert_array_equal(got[k], exp[k], err_msg=k)


def test_plan_rows_of_a_bad_page_have_no_slot(gpu):
    P = 16
    table = np.array([[99, -1], [1, -1]])
    free = np.array([0, 77, -1, -1])                       # 77 is no page
    p = Plan(gpu, [3, 16], None, [2, 2], table, P, free, 2, 4, 4, False)
    got = p.run()
    np.testing.assert_array_equal(got["slot"], [-1, -1, -1, -1])
    np.testing.assert_array_equal(got["table"], [[99, -1], [1, 77]])


# ------------------------------------------------------------------ append

def _rotated(x, cs):
    """x [n, heads, D], cs [n, D/2, 2], each product rounded in fp32."""
    h = x.shape[-1] // 2
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    return np.concatenate([x[..., :h] * c - x[..., h:] * s, x[..., :h] * s + x[..., h:] * c], -1)


@pytest.mark.parametrize("T,H,Hk,D,gs,P,rope,q", [
    (5, 32, 8, 128, 128, 16, True, True), (1, 1, 1, 32, 32, 16, True, True), (33, 12, 12, 64, 32, 64, True, True),
    (7, 28, 4, 128, 64, 32, False, True), (9, 0, 3, 96, 48, 16, True, False), (4, 7, 9, 256, 2, 16, True, True),
    (130, 16, 2, 96, 96, 256, True, True), (3, 5, 17, 160, 20, 16, True, True), (6, 8, 1, 64, 64, 16, True, False)])
def test_append_and_gather(gpu, oracle, T, H, Hk, D, gs, P, rope, q):
    rng = np.random.default_rng(T + D + gs)
    layers, layer, pages, ldq = 2, 1, R.pages_of(T, P) + 3, (H + 2 * Hk) * D + 4
    pool = R.Pool(layers, pages, P, Hk, D, gs)
    cache = pool.upload(gpu)
    x = rng.normal(size=(T, ldq)).astype(np.float32)
    x[0, H * D:H * D + D] = 0.0                            # a key of zeros: scale 1
    pos = rng.integers(0, 50, T)
    slot = rng.permutation(pages * P)[:T]
    skip = set()
    if T > 3:
        slot[1], slot[2] = -1, pages * P                   # padding, a bad slot
        skip |= {1, 2}
        if rope:
            pos[3] = 50                                    # past the rotary table
            skip.add(3)
    cs = rng.normal(size=(50, D // 2, 2)).astype(np.float32)
    dq = _dev(gpu, np.full((T, max(H, 1), D), 3.0), np.float32)
    dx, dcs, dslot, dpos = _dev(gpu, x, np.float32), _dev(gpu, cs, np.float32), _dev(gpu, slot), _dev(gpu, pos)
    st = CgxPagedStep(seqs=1, rows=T, max_rows=0, table_ld=1)
    st.row_slot, st.row_pos = dslot.ptr, dpos.ptr
    rc = gpu.cgx_kv_paged_append_dev(C.byref(cache), layer, C.byref(st), dx.ptr, ldq, H,
                                     dcs.ptr if rope else None, 50 if rope else 0, dq.ptr if q else None)
    assert rc == 0 and gpu.cgx_synchronize() == 0, last_error(gpu)
    h = x[:, :(H + 2 * Hk) * D].reshape(T, H + 2 * Hk, D)
    qk = h[:, :H + Hk]
    at = np.minimum(pos, 49)
    turned = _rotated(qk, cs[at]) if rope else qk
    live = [t for t in range(T) if t not in skip]
    got_q = dq.numpy(np.float32, (T, max(H, 1), D))
    for t in range(T):
        exp = turned[t, :H] if q and t in live else np.full((max(H, 1), D), 3.0, np.float32)
        np.testing.assert_array_equal(got_q[t, :len(exp)], exp)
    kv = []
    for y in (np.ascontiguousarray(turned[:, H:]), np.ascontiguousarray(h[:, H + Hk:])):
        # the contiguous cache's quantiser in the oracle: flat groups of gs
        data, scales = oracle_lib.oracle_quantize(oracle, y.reshape(T * Hk, D), gs)
        nib = np.stack([data & 15, data >> 4], -1).reshape(T, Hk, D).astype(np.int64)
        code, s = np.where(nib >= 8, nib - 16, nib), scales.reshape(T, Hk, D // gs)
        c2, s2 = R.quantise(y, gs)
        np.testing.assert_array_equal(code, c2)
        np.testing.assert_array_equal(s, s2)
        kv += [code, s]
    for t in live:
        pool.put(layer, int(slot[t]), kv[0][t], kv[1][t], kv[2][t], kv[3][t])
    for got, exp in zip(pool.download(), (pool.k, pool.v, pool.ks, pool.vs)):
        np.testing.assert_array_equal(got, exp)            # nothing else written, NaN in place
    dk, dv = (_dev(gpu, np.full((T, Hk, D), 9.0), np.float32) for _ in range(2))
    assert gpu.cgx_kv_paged_gather_dev(C.byref(cache), layer, dslot.ptr, T, dk.ptr, dv.ptr) == 0
    assert gpu.cgx_synchronize() == 0, last_error(gpu)
    for d, code, s in ((dk, kv[0], kv[1]), (dv, kv[2], kv[3])):
        got = d.numpy(np.float32, (T, Hk, D))
        exp = R.values(code, s).astype(np.float32)         # a code times a scale, rounded once
        for t in live:
            np.testing.assert_array_equal(got[t], exp[t])
        for t in skip & {1, 2}:
            np.testing.assert_array_equal(got[t], 0.0)


def test_append_writes_what_the_contiguous_cache_holds(gpu):
    """The fused contiguous form and the paged one give the same values for the same rows."""
    rng = np.random.default_rng(3)
    T, H, Hk, D, P = 6, 8, 2, 128, 16
    x = rng.normal(size=(T, (H + 2 * Hk) * D)).astype(np.float32)
    dx = _dev(gpu, x, np.float32)
    rope = DeviceArray(gpu, T * D * 4)
    assert gpu.cgx_rope_table_dev(T, D, 0, 10000.0, rope.ptr) == 0
    flat = gpu.cg_kv_cache_int4_new(1, 32, Hk, D, D)
    o = DeviceArray(gpu, T * H * D * 4)
    assert gpu.cgx_attention_rope_append_dev(dx.ptr, x.shape[1], rope.ptr, T, H, flat, 0, 0, o.ptr) == 0
    assert gpu.cgx_kv_cache_int4_set_len(flat, T) == 0
    cache = gpu.cgx_kv_paged_int4_new(1, 3, P, Hk, D, D)
    slot, pos = _dev(gpu, np.arange(T) + 20), _dev(gpu, np.arange(T))
    st = CgxPagedStep(seqs=1, rows=T, max_rows=0, table_ld=1)
    st.row_slot, st.row_pos = slot.ptr, pos.ptr
    assert gpu.cgx_kv_paged_append_dev(cache, 0, C.byref(st), dx.ptr, x.shape[1], H, rope.ptr, T, None) == 0
    k, v = DeviceArray(gpu, T * Hk * D * 4), DeviceArray(gpu, T * Hk * D * 4)
    assert gpu.cgx_kv_paged_gather_dev(cache, 0, slot.ptr, T, k.ptr, v.ptr) == 0
    from gpu_util import device_tensor, tensor_np
    tk, tv = (device_tensor(gpu, np.zeros((T, Hk, D), np.float32)) for _ in range(2))
    gpu.cg_kv_cache_int4_get(flat, 0, tk, tv)
    assert gpu.cgx_synchronize() == 0
    np.testing.assert_array_equal(k.numpy(np.float32, (T, Hk, D)), tensor_np(gpu, tk))
    np.testing.assert_array_equal(v.numpy(np.float32, (T, Hk, D)), tensor_np(gpu, tv))
    for t in (tk, tv):
        gpu.cg_tensor_free(t)
    gpu.cg_kv_cache_int4_free(flat)
    gpu.cgx_kv_paged_int4_free(cache)


# --------------------------------------------------------------- attention

def _check(b, got, ref, rows=None):
    (o, ls), (O, L, A, F) = got, ref
    n = int(b.begin[-1])
    d = np.abs(o[:n] - O[:n])
    assert np.all(np.isfinite(o[:n]))
    bad = d > TOL * A[:n] + F[:n] + 1e-37
    assert not bad.any(), (float((d / np.maximum(A[:n], 1e-300)).max()), np.argwhere(bad)[:4].tolist())
    np.testing.assert_array_equal(o[n:], 7.0)              # rows behind the last sequence
    if ls is not None:
        e = L[:n]
        fin = np.isfinite(e)
        np.testing.assert_array_equal(ls[:n][~fin], e[~fin])
        assert np.all(np.abs(ls[:n][fin] - e[fin]) <= TOL * (1 + np.abs(e[fin])))
        np.testing.assert_array_equal(ls[n:], 7.0)


HEADS = [(4, 1, 32, 32), (8, 2, 64, 64), (12, 12, 64, 32), (16, 2, 96, 96), (6, 2, 96, 32), (8, 2, 128, 128),
         (28, 4, 128, 64), (32, 8, 128, 32), (32, 1, 128, 128), (4, 2, 96, 48), (2, 1, 160, 160),
         (6, 3, 256, 128), (3, 1, 64, 2)]


@pytest.mark.parametrize("H,Hk,D,gs", HEADS)
@pytest.mark.parametrize("kv,rows,P", [
    ([1], [1], 16), ([300], [5], 16), ([17, 1, 256, 0, 33, 640], [1, 1, 3, 0, 0, 8], 16),
    ([70, 129], [70, 40], 64), ([15, 16, 17, 31, 32, 33, 63, 64, 65], [2, 1, 5, 1, 3, 7, 1, 4, 1], 32)])
def test_attention_chain(gpu, H, Hk, D, gs, kv, rows, P):
    rng = np.random.default_rng(D + gs + sum(kv))
    b = R.Batch(gpu, rng, kv, rows, P, H, Hk, D, gs, layer=1, layers=2, pad=3).bind()
    _check(b, b.attend(), b.reference())


@pytest.mark.parametrize("H,Hk,D,gs", [(32, 8, 128, 128), (12, 12, 64, 32), (16, 2, 96, 96)])
@pytest.mark.parametrize("kv,rows,P", [
    ([2100], [1], 16), ([3000], [5], 256), ([1029], [509], 16), ([700, 40, 333, 1500], [130, 1, 65, 2], 128)])
def test_attention_long_and_prompts(gpu, H, Hk, D, gs, kv, rows, P):
    rng = np.random.default_rng(7 + sum(kv))
    b = R.Batch(gpu, rng, kv, rows, P, H, Hk, D, gs, pad=2).bind()
    ref = b.reference()
    _check(b, b.attend(), ref)
    # the same without lse and with the rows' bound given
    _check(b, b.attend(lse=False, max_rows=max(rows)), ref)


def _tree(rng, n, tw=None):
    tw = n if tw is None else tw
    out = []
    for i in range(n):
        me = tw - n + i
        bits = int(rng.integers(0, 2**62)) & ((1 << max(0, min(me, 64))) - 1)
        out.append(bits | (1 << me if me < 64 else 0))
    return out


@pytest.mark.parametrize("H,Hk,D,gs", [(8, 2, 128, 128), (12, 12, 64, 32), (4, 2, 96, 48), (32, 8, 128, 32)])
@pytest.mark.parametrize("kv,rows,P,window", [
    ([80], [64], 16, False), ([7, 200, 64, 9], [7, 13, 64, 1], 16, False), ([90, 300, 33], [5, 30, 1], 32, True)])
def test_attention_trees(gpu, H, Hk, D, gs, kv, rows, P, window):
    rng = np.random.default_rng(D + sum(rows))
    b = R.Batch(gpu, rng, kv, rows, P, H, Hk, D, gs, pad=1).bind()
    tw = [min(64, k, r + 17) for k, r in zip(kv, rows)] if window else None
    anc = []
    for i, n in enumerate(rows):
        anc += _tree(rng, n, tw[i] if window else None)
    anc[0] = 0                                             # sees nothing of the tree
    anc += [0] * (b.T - len(anc))
    _check(b, b.attend(anc=anc, tree_len=tw), b.reference(anc=anc, tree_len=tw))


def test_attention_rows_that_see_nothing(gpu):
    """Rows in front of the first key (more rows than keys), an all-hidden tree, an empty sequence."""
    rng = np.random.default_rng(1)
    b = R.Batch(gpu, rng, [3, 5, 0], [6, 5, 2], 16, 8, 2, 128, 128, pad=1).bind()
    ref = b.reference()
    assert np.isneginf(ref[1][:3]).all() and np.isneginf(ref[1][11:13]).all()
    _check(b, b.attend(), ref)
    anc = [0] * b.T
    got = b.attend(anc=anc)
    _check(b, got, b.reference(anc=anc))
    assert not got[0][:13].any()


def test_attention_hidden_keys_hold_anything(gpu):
    """NaN and infinite scales of keys that a row does not see do not reach it."""
    rng = np.random.default_rng(2)
    kv, rows, P = [70, 40], [20, 9], 16
    b = R.Batch(gpu, rng, kv, rows, P, 8, 2, 128, 128)
    last = b.table[0, 69 // P] * P + 69 % P                # seen by the last row alone
    for a, x in ((b.pool.ks, np.nan), (b.pool.vs, np.inf)):
        a[0, last // P, :, last % P] = x
    b.bind()
    ref = b.reference()
    o, ls = b.attend()
    keep = np.r_[0:19, 20:29]
    assert np.all(np.isfinite(o[keep]))
    assert np.all(np.abs(o[keep] - ref[0][keep]) <= TOL * ref[2][keep])
    assert not np.isfinite(o[19]).any()


def test_attention_pages_outside_the_pool_are_not_seen(gpu):
    rng = np.random.default_rng(4)
    kv, rows, P = [100, 20, 600], [4, 20, 3], 16
    b = R.Batch(gpu, rng, kv, rows, P, 8, 2, 128, 128)
    seen = [np.ones(n, bool) for n in kv]
    b.table[0, 2], b.table[1, 0], b.table[2, 5] = -1, 2**31 - 1, b.pool.dims[1]
    seen[0][32:48] = seen[1][0:16] = seen[2][80:96] = False
    b.bind()
    _check(b, b.attend(), b.reference(seen=seen))


def test_attention_lengths_past_the_table_are_cut(gpu):
    """A length or row offset that no table or row array backs reads and writes nothing outside them."""
    rng = np.random.default_rng(6)
    b = R.Batch(gpu, rng, [40, 30], [2, 1], 16, 8, 2, 128, 128, pad=4).bind()
    b.d["kv"].upload(np.array([2**31 - 1, -5], np.int32))
    o, ls = b.attend()
    assert np.all(o[3:] == 7.0) and not o[2].any() and np.isneginf(ls[2]).all()
    b.d["kv"].upload(np.array([40, 30], np.int32))
    # the row offsets say whose a row is: here all rows from 2 on are the second sequence's
    b.d["begin"].upload(np.array([0, 2, 2**31 - 1], np.int32))
    o, _ = b.attend(lse=False)
    assert np.all(np.isfinite(o))
    b.d["begin"].upload(np.array([-7, -5, -1], np.int32))
    o, _ = b.attend(lse=False)
    assert np.all(o == 7.0)


@pytest.mark.parametrize("which", ["k", "v", "q_small", "q_large"])
def test_attention_of_far_apart_scales(gpu, which):
    """Positions whose scales lie 2^60 apart, queries far from 1."""
    rng = np.random.default_rng(8)
    far = lambda r, n: 2.0 ** r.integers(-30, 31, n)       # noqa: E731
    kw = {"k": dict(kscale=lambda r, n: 2.0 ** r.integers(-30, 1, n)), "v": dict(vscale=far),
          "q_small": dict(qscale=1e-30, kscale=lambda r, n: np.full(n, 1e30)),
          "q_large": dict(qscale=1e30, kscale=lambda r, n: np.full(n, 1e-30))}[which]
    b = R.Batch(gpu, rng, [400, 77, 20], [5, 1, 20], 16, 8, 2, 128, 128, **kw)
    b.bind()
    _check(b, b.attend(), b.reference())


def test_attention_split_of_one_dominant_key(gpu):
    """One key far from the query's position takes all weight, and its values are small."""
    rng = np.random.default_rng(9)
    b = R.Batch(gpu, rng, [5000], [1], 16, 4, 1, 128, 128,
                vscale=lambda r, n: np.where(np.arange(n) == 123, 2.0 ** -25, 1.0))
    b.q[0, :] = 8.0 * b.K[0][123, 0].astype(np.float32)
    b.bind()
    _check(b, b.attend(), b.reference())


# ------------------------------------------------------- a step as it is used

class Serving:
    """Tables, append, attention and log probabilities of a batch of requests, everything on the device."""

    def __init__(self, lib, rng, B, P, H, Hk, D, V, ld, rows):
        self.lib, self.B, self.P, self.H, self.Hk, self.D, self.V, self.T = lib, B, P, H, Hk, D, V, rows
        self.pages = B * ld
        self.cache = lib.cgx_kv_paged_int4_new(1, self.pages, P, Hk, D, D)
        assert self.cache, last_error(lib)
        z = lambda n: _dev(lib, np.zeros(n))               # noqa: E731
        self.d = dict(old=z(B), keep=z(B), new=z(B), begin=z(B + 1), seq=z(rows), pos=z(rows), slot=z(rows),
                      kv=z(B), status=z(4), count=_dev(lib, [self.pages]), left=z(1),
                      free=_dev(lib, rng.permutation(self.pages)), table=_dev(lib, np.full((B, ld), -1)))
        st = CgxPagedStep(seqs=B, rows=rows, max_rows=0, table_ld=ld)
        st.kv_old, st.kv_keep, st.rows_new, st.table = (self.d[k].ptr for k in ("old", "keep", "new", "table"))
        st.row_begin, st.row_seq, st.row_pos, st.row_slot, st.kv_len, st.status = (
            self.d[k].ptr for k in ("begin", "seq", "pos", "slot", "kv", "status"))
        self.step = st
        self.rope = DeviceArray(lib, ld * P * D * 4)
        assert lib.cgx_rope_table_dev(ld * P, D, 0, 10000.0, self.rope.ptr) == 0
        f = lambda *n: DeviceArray(lib, int(np.prod(n)) * 4)   # noqa: E731
        self.x, self.q, self.o = f(rows, (H + 2 * Hk) * D), f(rows, H, D), f(rows, H, D)
        self.logits, self.tok = f(rows, V), z(rows)
        self.lp, self.rank, self.ent, self.top, self.top_lp = f(rows), z(rows), f(rows), z(rows * 3), f(rows, 3)
        n = max(lib.cgx_attention_paged_ws(self.cache, C.byref(st), H), lib.cgx_token_logprobs_ws(rows, V, 3))
        self.ws = DeviceArray(lib, n)

    def issue(self):
        lib, s = self.lib, C.byref(self.step)
        return (lib.cgx_paged_plan_dev(s, self.P, self.pages, self.d["free"].ptr, self.d["count"].ptr,
                                       self.d["left"].ptr) or
                lib.cgx_kv_paged_append_dev(self.cache, 0, s, self.x.ptr, (self.H + 2 * self.Hk) * self.D, self.H,
                                            self.rope.ptr, self.step.table_ld * self.P, self.q.ptr) or
                lib.cgx_attention_paged_dev(self.cache, 0, s, self.q.ptr, self.H, None, None, self.o.ptr, None,
                                            self.ws.ptr, self.ws.nbytes) or
                lib.cgx_token_logprobs_dev(self.logits.ptr, self.V, self.T, self.V, self.tok.ptr, 3, self.lp.ptr,
                                           self.rank.ptr, self.ent.ptr, self.top.ptr, self.top_lp.ptr, self.ws.ptr,
                                           self.ws.nbytes))


def test_serving_steps_eager_and_captured(gpu):
    """Requests of different lengths through several steps with rollbacks: a captured step replayed with eager
    work and synchronisation in between, against the same history in 64 bits, and against eager steps bit for bit."""
    B, P, H, Hk, D, V, ld, rows = 5, 16, 8, 2, 128, 1000, 6, 24
    both = [Serving(gpu, np.random.default_rng(11), B, P, H, Hk, D, V, ld, rows) for _ in range(2)]
    rng = np.random.default_rng(12)
    g = None
    hist_k, hist_v = [[] for _ in range(B)], [[] for _ in range(B)]
    rope = both[0].rope.numpy(np.float32, (ld * P, D // 2, 2))
    kv = np.zeros(B, int)
    for step in range(6):
        keep = kv - np.minimum(kv, rng.integers(0, 4, B)) if step else kv
        if step == 4:
            keep[1] = 0                                    # a request ends, another takes its place
        new = rng.integers(0, 6, B)
        if step == 0:
            new = np.array([1, 9, 4, 0, 7])
        if step == 5:
            new[:] = 0                                     # a step without rows
        x = rng.normal(size=(rows, (H + 2 * Hk) * D)).astype(np.float32)
        logits = rng.normal(size=(rows, V)).astype(np.float32) * 3
        tok = rng.integers(0, V, rows)
        for s in both:
            for k, a in (("old", kv), ("keep", keep), ("new", new)):
                s.d[k].upload(np.asarray(a, np.int32))
            if step:
                s.d["count"].upload(s.d["left"].numpy(np.int32, (1,)))
            s.x.upload(x)
            s.logits.upload(logits)
            s.tok.upload(tok.astype(np.int32))
            s.o.upload(np.full((rows, H, D), 7.0, np.float32))
        assert both[0].issue() == 0, last_error(gpu)
        assert gpu.cgx_synchronize() == 0
        if g is None:
            assert gpu.cgx_graph_begin() == 0
            rc = both[1].issue()
            g = gpu.cgx_graph_end()
            assert rc == 0 and g, last_error(gpu)
        assert gpu.cgx_graph_launch(g) == 0 and gpu.cgx_synchronize() == 0, last_error(gpu)
        T = int(new.sum())
        for name, n, t in (("o", rows * H * D, np.uint32), ("lp", rows, np.uint32), ("rank", rows, np.uint32),
                           ("ent", rows, np.uint32), ("top", rows * 3, np.uint32), ("top_lp", rows * 3, np.uint32)):
            a, b = (getattr(s, name).numpy(t, (n,)) for s in both)
            np.testing.assert_array_equal(a, b, err_msg=f"step {step} {name}")
        kv = keep + new
        np.testing.assert_array_equal(both[0].d["kv"].numpy(np.int32, (B,)), kv)
        o = both[0].o.numpy(np.float32, (rows, H, D))
        assert np.all(o[T:] == 7.0)
        hx = x.reshape(rows, H + 2 * Hk, D)
        t = 0
        for b in range(B):
            del hist_k[b][keep[b]:], hist_v[b][keep[b]:]
            for i in range(new[b]):
                y = hx[t + i:t + i + 1]
                cs = rope[keep[b] + i][None]
                hist_k[b].append(R.values(*R.quantise(_rotated(y[:, H:H + Hk], cs), D))[0])
                hist_v[b].append(R.values(*R.quantise(y[:, H + Hk:], D))[0])
                q = _rotated(y[:, :H], cs)[0].astype(np.float64)
                K, Vv = np.array(hist_k[b]), np.array(hist_v[b])
                for h in range(H):
                    sc = K[:, h // 4] @ q[h] / np.sqrt(D)
                    p = np.exp(sc - sc.max())
                    p /= p.sum()
                    assert np.all(np.abs(o[t + i, h] - p @ Vv[:, h // 4]) <= TOL * (p @ np.abs(Vv[:, h // 4])))
            t += new[b]
    assert gpu.cgx_graph_free(g) == 0
    for s in both:
        gpu.cgx_kv_paged_int4_free(s.cache)
