"""The paged cache's steps in plain numpy: tables by loops, the page layout, attention in 64 bits."""
from __future__ import annotations

import ctypes as C

import numpy as np

from cogito_amd.capi import CgxKvPagedInt4, CgxPagedStep, DeviceArray, last_error


def pages_of(n, P):
    return -(-int(n) // P)


def plan(old, keep, new, table_old, P, free, count, rows, ld, num_pages, max_rows=0):
    """(refusal bits, dict of outputs) of one planned step; table: the new table with -1 past each sequence's pages."""
    B = len(old)
    bits = 0
    for b in range(B):
        if keep[b] < 0 or keep[b] > old[b] or new[b] < 0:
            bits |= 1
        elif old[b] > ld * P or keep[b] + new[b] > ld * P:
            bits |= 2
        elif new[b] > rows or (max_rows and new[b] > max_rows):
            bits |= 4
    ok = [b for b in range(B) if not (keep[b] < 0 or keep[b] > old[b] or new[b] < 0 or
                                      old[b] > ld * P or keep[b] + new[b] > ld * P or
                                      new[b] > rows or (max_rows and new[b] > max_rows))]
    if sum(int(new[b]) for b in ok) > rows:
        bits |= 4
    give = [(b, j) for b in ok for j in range(pages_of(keep[b] + new[b], P), pages_of(old[b], P))]
    take = [(b, j) for b in ok for j in range(pages_of(old[b], P), pages_of(keep[b] + new[b], P))]
    if count < 0 or count > num_pages or count + len(give) > num_pages:
        bits |= 16
    elif len(take) > count + len(give):
        bits |= 8
    seq, pos, slot = (np.full(rows, -1, np.int64) for _ in range(3))
    begin = np.zeros(B + 1, np.int64)
    if bits:
        return bits, dict(begin=begin, seq=seq, pos=pos, slot=slot, kv=np.array(old), left=count,
                          free=np.array(free), table=np.array(table_old), status=[bits, 0, 0, 0])
    stack = list(free[:count]) + [table_old[b][j] for b, j in give]
    table = np.full((B, ld), -1, np.int64)
    for b in range(B):
        for j in range(min(pages_of(old[b], P), pages_of(keep[b] + new[b], P))):
            table[b, j] = table_old[b][j]
    for b, j in take:
        table[b, j] = stack.pop()
    out_free = np.array(free)
    for at in range(count, len(stack)):
        out_free[at] = stack[at]
    t = 0
    for b in range(B):
        begin[b] = t
        for i in range(new[b]):
            p = keep[b] + i
            page = table[b, p // P]
            seq[t], pos[t] = b, p
            slot[t] = page * P + p % P if 0 <= page < num_pages else -1
            t += 1
    begin[B] = t
    return 0, dict(begin=begin, seq=seq, pos=pos, slot=slot, kv=np.array(keep) + np.array(new),
                   left=len(stack), free=out_free, table=table,
                   status=[0, t, len(take), len(give)])


# ------------------------------------------------------------------ layout

def quantise(x, gs):
    """Codes (float) and fp32 scales of x [..., D] by the cache's rule, every step in 32 bits."""
    t = np.ascontiguousarray(x, np.float32).reshape(*x.shape[:-1], x.shape[-1] // gs, gs)
    s = (np.abs(t).max(-1) / np.float32(7)).astype(np.float32)
    s = np.where(s < np.float32(1e-8), np.float32(1), s)
    r = (t / s[..., None]).astype(np.float32).astype(np.float64)
    code = np.clip(np.sign(r) * np.floor(np.abs(r) + 0.5), -8, 7)
    return code.reshape(x.shape), s


def values(code, s):
    D = code.shape[-1]
    return (code.reshape(*code.shape[:-1], s.shape[-1], D // s.shape[-1]) *
            s.astype(np.float64)[..., None]).reshape(*code.shape[:-1], D)


class Pool:
    """One layer stack's pages on the host in the library's layout; positions nobody wrote hold NaN scales and 0xAB bytes."""

    def __init__(self, layers, pages, P, Hk, D, gs):
        self.dims = (layers, pages, P, Hk, D, gs)
        self.k = np.full((layers, pages, Hk, P, D // 2), 0xAB, np.uint8)
        self.v = np.full((layers, pages, Hk, P // 16, 16, 16, D // 32), 0xAB, np.uint8)
        self.ks = np.full((layers, pages, Hk, P, D // gs), np.nan, np.float32)
        self.vs = np.full((layers, pages, Hk, P, D // gs), np.nan, np.float32)

    def put(self, layer, slot, kc, ks, vc, vs):
        """Codes [Hk, D] and scales of one position."""
        _, _, P, Hk, D, _ = self.dims
        pg, at = slot // P, slot % P
        nib = lambda c: ((c[:, 0::2].astype(int) & 15) | ((c[:, 1::2].astype(int) & 15) << 4)).astype(np.uint8)  # noqa: E731
        self.k[layer, pg, :, at] = nib(kc)
        self.v[layer, pg, :, at // 16, :, at % 16] = nib(vc).reshape(Hk, 16, D // 32)
        self.ks[layer, pg, :, at] = ks
        self.vs[layer, pg, :, at] = vs

    def upload(self, lib):
        layers, pages, P, Hk, D, gs = self.dims
        self.dev = [DeviceArray.from_numpy(lib, a) for a in (self.k, self.v, self.ks, self.vs)]
        c = CgxKvPagedInt4(num_layers=layers, num_pages=pages, page_size=P, n_heads=Hk, head_dim=D,
                           group_size=gs)
        c.k_pages, c.v_pages, c.k_scales, c.v_scales = (d.ptr for d in self.dev)
        return c

    def download(self):
        return [d.numpy(a.dtype, a.shape) for d, a in zip(self.dev, (self.k, self.v, self.ks, self.vs))]


class Batch:
    """Sequences with random keys and values in a pool, their table and row offsets on the device."""

    def __init__(self, lib, rng, kv, rows, P, H, Hk, D, gs, layer=0, layers=1, pad=0, kscale=None,
                 vscale=None, qscale=1.0):
        self.lib, self.kv, self.rows, self.P = lib, list(kv), list(rows), P
        self.H, self.Hk, self.D, self.gs, self.layer = H, Hk, D, gs, layer
        B = len(kv)
        need = [pages_of(n, P) for n in kv]
        pages = sum(need) + 3
        ld = max(need + [1]) + 1
        order = rng.permutation(pages)
        self.table = np.full((B, ld), -1, np.int32)
        at = 0
        for b in range(B):
            self.table[b, :need[b]] = order[at:at + need[b]]
            at += need[b]
        self.pool = Pool(layers, pages, P, Hk, D, gs)
        self.K, self.V, self.vs = [], [], []
        for b in range(B):
            n = kv[b]
            k = rng.normal(size=(n, Hk, D)).astype(np.float32)
            v = rng.normal(size=(n, Hk, D)).astype(np.float32)
            kc, ks = quantise(k, gs)
            vc, vs = quantise(v, gs)
            if kscale is not None:                     # scales of any size, also below the quantiser's floor
                ks = (ks * kscale(rng, n)[:, None, None]).astype(np.float32)
            if vscale is not None:
                vs = (vs * vscale(rng, n)[:, None, None]).astype(np.float32)
            for j in range(n):
                slot = int(self.table[b, j // P]) * P + j % P
                self.pool.put(layer, slot, kc[j], ks[j], vc[j], vs[j])
            self.K.append(values(kc, ks))
            self.V.append(values(vc, vs))
            self.vs.append(vs.astype(np.float64))
        self.begin = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.T = int(self.begin[-1]) + pad
        self.seq = np.full(self.T, -1, np.int32)
        self.seq[:self.begin[-1]] = np.repeat(np.arange(B), rows)
        self.q = (rng.normal(size=(self.T, H, D)) * qscale).astype(np.float32)

    def bind(self):
        lib = self.lib
        self.cache = self.pool.upload(lib)
        B = len(self.kv)
        up = lambda a, t=np.int32: DeviceArray.from_numpy(lib, np.asarray(a, t))  # noqa: E731
        self.d = dict(table=up(self.table), begin=up(self.begin), seq=up(self.seq), kv=up(self.kv),
                      q=DeviceArray.from_numpy(lib, self.q))
        st = CgxPagedStep(seqs=B, rows=self.T, max_rows=0, table_ld=self.table.shape[1])
        st.table, st.row_begin, st.row_seq = self.d["table"].ptr, self.d["begin"].ptr, self.d["seq"].ptr
        st.kv_len = self.d["kv"].ptr
        self.step = st
        return self

    def attend(self, anc=None, tree_len=None, lse=True, fill=7.0, max_rows=0):
        """(O, lse) of the library, both started at `fill`."""
        lib, T, H, D = self.lib, self.T, self.H, self.D
        o = DeviceArray.from_numpy(lib, np.full(T * H * D + 512, fill, np.float32))     # guard words behind
        ls = DeviceArray.from_numpy(lib, np.full((T, H), fill, np.float32)) if lse else None
        da = DeviceArray.from_numpy(lib, np.asarray(anc, np.uint64)) if anc is not None else None
        dl = DeviceArray.from_numpy(lib, np.asarray(tree_len, np.int32)) if tree_len is not None else None
        self.step.max_rows = max_rows
        need = lib.cgx_attention_paged_ws(C.byref(self.cache), C.byref(self.step), H)
        # guard words behind the workspace
        ws = DeviceArray.from_numpy(lib, np.full(need + 256, 0xC3, np.uint8))
        rc = lib.cgx_attention_paged_dev(C.byref(self.cache), self.layer, C.byref(self.step),
                                         self.d["q"].ptr, H, da.ptr if da else None,
                                         dl.ptr if dl else None, o.ptr, ls.ptr if ls else None,
                                         ws.ptr, need)
        assert rc == 0, last_error(lib)
        assert lib.cgx_synchronize() == 0, last_error(lib)
        assert np.all(ws.numpy(np.uint8, (need + 256,))[need:] == 0xC3)
        assert np.all(o.numpy(np.float32, (T * H * D + 512,))[T * H * D:] == fill)
        return o.numpy(np.float32, (T, H, D)), ls.numpy(np.float32, (T, H)) if lse else None

    def visible(self, b, anc=None, tree_len=None, seen=None):
        """[rows, kv] of sequence b."""
        L, n = self.kv[b], self.rows[b]
        j = np.arange(L)
        if anc is None:
            vis = j[None] <= (L - n + np.arange(n))[:, None]
        else:
            w = min(max(tree_len[b] if tree_len is not None else n, 0), L)
            base = L - w
            d = np.clip(j - base, 0, 63).astype(np.uint64)
            bits = np.asarray(anc, np.uint64)[self.begin[b]:self.begin[b + 1], None]
            vis = (j < base)[None] | ((((bits >> d[None]) & np.uint64(1)) > 0) & (j - base < 64)[None])
        if seen is not None:
            vis = vis & seen[b][None, :L]
        return vis

    def reference(self, anc=None, tree_len=None, seen=None):
        """O, lse, A = sum_j p_j |v_j| (the scale of O's rounding errors) and N 2^-36 max_j p_j s_j, in 64 bits."""
        T, H, Hk, D = self.T, self.H, self.Hk, self.D
        O, A, F, ls = np.zeros((T, H, D)), np.zeros((T, H, D)), np.zeros((T, H, D)), np.full((T, H), -np.inf)
        for b in range(len(self.kv)):
            r0, r1 = self.begin[b], self.begin[b + 1]
            if r1 == r0 or self.kv[b] == 0:
                continue
            vis = self.visible(b, anc, tree_len, seen)
            for h in range(H):
                hk = h // (H // Hk)
                s = self.q[r0:r1, h].astype(np.float64) @ self.K[b][:, hk].T / np.sqrt(D)
                s = np.where(vis, s, -np.inf)
                m = s.max(1, keepdims=True)
                m = np.where(np.isfinite(m), m, 0.0)
                e = np.exp(s - m)
                z = e.sum(1, keepdims=True)
                p = e / np.where(z > 0, z, 1.0)
                O[r0:r1, h] = p @ self.V[b][:, hk]
                A[r0:r1, h] = p @ np.abs(self.V[b][:, hk])
                w = np.nan_to_num(p[:, :, None] * self.vs[b][None, :, hk], nan=0.0).max(1)
                F[r0:r1, h] = np.repeat(w, self.gs, -1) * self.kv[b] * 2.0 ** -36
                with np.errstate(divide="ignore"):
                    ls[r0:r1, h] = (m + np.log(z))[:, 0]
        return O, ls, A, F
