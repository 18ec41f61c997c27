"""Operators of a serving step over a paged INT4 KV cache, in plain form and as the library's calls.

A step of a server that verifies drafts for many requests of different lengths:

  tables     pages that a step's new rows need, taken from a stack of free pages on which the pages of
             rejected drafts and ended requests go back first: block tables, slot of every row, row
             offsets (cgx_paged_plan_dev)
  append     rotary positions and the 4-bit append of the new rows into their slots
             (cgx_kv_paged_append_dev), read back as values (cgx_kv_paged_gather_dev)
  attention  the new rows over each sequence's pages (cgx_attention_paged_dev), chain or tree masks
  logprobs   log probability, rank, entropy and top alternatives of the emitted tokens
             (cgx_token_logprobs_dev)

Packed pages (the layout of cgx_kv_paged_int4, one layer): K bytes [page][head][position][D/2], V bytes
[page][head][position/16][16][position%16][D/32], that is D/16 neighbouring dimensions of 16 positions
side by side; scales [page][head][position][D/group].  A byte holds two values, the even one in its low
nibble, in two's complement.

Sizes are those of the benchmark's stacks (32 query heads over 8 KV heads of 128, 12 heads of 64,
vocabularies of 32000, 50257 and 128256, gamma 4) and of contexts up to 131072; `draw` spreads over the ranges
around them.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False


# ------------------------------------------------------------------ cases

def _tables(B, ctx, rows, page, rollback, **name):
    return dict(name, kind="tables", B=B, ctx=ctx, rows=rows, page=page, rollback=rollback)


def _append(B, ctx, rows, page, H, Hk, D, gs, **name):
    return dict(name, kind="append", B=B, ctx=ctx, rows=rows, page=page, H=H, Hk=Hk, D=D, gs=gs)


def _attention(B, ctx, rows, prompts, chunk, page, H, Hk, D, gs, tree, lse, **name):
    return dict(name, kind="attention", B=B, ctx=ctx, rows=rows, prompts=prompts, chunk=chunk,
                page=page, H=H, Hk=Hk, D=D, gs=gs, tree=tree, lse=lse)


def _logprobs(rows, V, top, masked, **name):
    return dict(name, kind="logprobs", rows=rows, V=V, top=top, masked=masked)


def listed():
    return [
        # 64 requests, each with up to gamma + 1 rows, after the rejected
        # drafts of the last step gave their pages back: latency
        _tables(64, 4096, 5, 16, True, name="tables_verify"),
        # a large batch of admitted prompts of different lengths
        _tables(256, 1024, 381, 64, False, name="tables_prompts"),
        # one chain of gamma 4 and the bonus row: the smallest append
        _append(1, 4096, 5, 16, 32, 8, 128, 128, name="append_verify"),
        # 64 requests verified together
        _append(64, 4096, 5, 16, 32, 8, 128, 128, name="append_batch"),
        # a prompt chunk of an odd length, one scale per 32 dimensions
        _append(1, 2048, 2039, 64, 12, 12, 64, 32, name="append_prompt"),
        # one chain verified at context 4096: latency
        _attention(1, 4096, 5, 0, 0, 16, 32, 8, 128, 128, False, False, name="attention_verify"),
        # 64 requests of ragged lengths, one decoded token each
        _attention(64, 4096, 1, 0, 0, 16, 32, 8, 128, 128, False, False, name="attention_decode"),
        # one token over a very long context: the split over the key axis
        _attention(1, 131071, 1, 0, 0, 256, 32, 8, 128, 128, False, True, name="attention_long"),
        # a prompt chunk of an odd length after 2048 cached tokens
        _attention(1, 2048, 0, 1, 509, 16, 32, 8, 128, 128, False, False, name="attention_prompt"),
        # draft trees of ragged requests of the small decoder, scales per 32
        # dimensions: odd sizes, pages that end inside a tile
        _attention(13, 3001, 37, 0, 0, 32, 12, 12, 64, 32, True, True, name="attention_trees"),
        # the emitted rows of one chain: latency
        _logprobs(5, 32000, 5, False, name="logprobs_verify"),
        # the rows of a scored prompt at the large vocabulary, 20 alternatives
        _logprobs(301, 128256, 20, False, name="logprobs_prompt"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    """Query heads, KV heads, head_dim and values per scale."""
    H, Hk, D = rng.choice([(32, 8, 128), (32, 8, 128), (12, 12, 64), (28, 4, 128), (8, 1, 64),
                           (16, 2, 96), (16, 16, 128), (8, 8, 32)])
    return H, Hk, D, rng.choice([D, D, D, 32])


def draw(rng):
    kind = rng.choice(["tables", "append", "attention", "attention", "attention", "logprobs"])
    page = rng.choice([16, 16, 32, 64, 128, 256])
    if kind == "tables":
        B = _log_int(rng, 1, 512)
        rollback = rng.random() < 0.5
        rows = rng.choice([1, 2, 5, 8]) if rollback else _log_int(rng, 1, 512)
        while B * rows > 65536:
            rows //= 2
        return _tables(B, _log_int(rng, 16, 8192), rows, page, rollback)
    if kind == "append":
        H, Hk, D, gs = _heads(rng)
        B = _log_int(rng, 1, 64)
        rows = _log_int(rng, 1, 2039)
        while rows > 1 and B * rows * (H + 2 * Hk) * D > 2039 * 36 * 64:
            rows //= 2
        return _append(B, _log_int(rng, 16, 4096), rows, page, H, Hk, D, gs)
    if kind == "attention":
        H, Hk, D, gs = _heads(rng)
        tree = rng.random() < 0.2
        prompts = 0 if tree else rng.choice([0, 0, 1, 2])
        B = max(prompts, _log_int(rng, 1, 64))
        rows = _log_int(rng, 2, 64) if tree else rng.choice([1, 1, 2, 5, 8])
        chunk = _log_int(rng, 32, 509) if prompts else 0
        ctx = _log_int(rng, 16, 8192) if B > 1 or rng.random() < 0.6 else _log_int(rng, 8192, 131071)
        while prompts > 1 and prompts * chunk * (ctx + chunk) * H * D > 509 * 2300 * 4096:
            prompts -= 1
        while chunk > 2 and prompts * chunk * (ctx + chunk) * H * D > 509 * 2300 * 4096:
            chunk //= 2
        while ctx > 16 and B * ctx * Hk * D > 64 * 4096 * 1024:
            ctx //= 2
        while B > 1 and B * max(rows, chunk) * ctx * H * D > 3 * 509 * 2300 * 4096:
            B -= 1
        while B == 1 and max(rows, chunk) * (ctx + chunk) * H * D > 509 * 2300 * 4096:
            ctx //= 2
        return _attention(max(B, prompts), ctx, rows, prompts, chunk, page, H, Hk, D, gs, tree,
                          rng.random() < 0.5)
    V = rng.choice([32000, 128256, 50257, _log_int(rng, 100, 128256)])
    rows = _log_int(rng, 1, 640)
    while rows > 1 and rows * V > 301 * 128256:
        rows //= 2
    return _logprobs(rows, V, rng.choice([0, 1, 5, 10, 20, 20, 32]), rng.random() < 0.3)


# ----------------------------------------------------------------- inputs

def _gen(seed, salt=0):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + salt)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _lengths(c):
    """Cached positions and new rows of each sequence (host): a batch of one has the case's own, a batch ragged ones. They are
    the case's, so that the outputs of two seeds have the same shapes."""
    r = np.random.RandomState((c["B"] * 1000003 + c["ctx"] * 8191 + c["rows"] * 131 + c["page"]) % (1 << 31))
    B, ctx, most = c["B"], c["ctx"], max(c["rows"], 1)
    old = np.array([ctx]) if B == 1 else r.randint(max(1, ctx // 8), ctx + 1, B)
    new = np.array([most]) if B == 1 else r.randint(1, most + 1, B)
    n = c.get("prompts", 0)
    if n:
        new[:n] = c["chunk"] if B == 1 else r.randint(c["chunk"] // 2 + 1, c["chunk"] + 1, n)
    return old.astype(np.int64), new.astype(np.int64)


def _pages_of(x, page):
    return -(-x // page)


def _batch(c, seed):
    """A batch whose rows have their slots: lengths after the step, block table with the pages in random order, row arrays."""
    old, new = _lengths(c)
    r = np.random.RandomState(seed % (1 << 31))
    page, B = c["page"], c["B"]
    kv = old + new
    need = _pages_of(kv, page)
    width, total = int(need.max()), int(need.sum())
    pages = total + 3                                  # some that no sequence holds
    table = np.full((B, width), -1, np.int64)
    table[np.arange(width) < need[:, None]] = r.permutation(pages)[:total]
    begin = np.concatenate([[0], np.cumsum(new)])
    seq = np.repeat(np.arange(B), new)
    pos = np.arange(begin[-1]) - begin[seq] + old[seq]
    slot = table[seq, pos // page] * page + pos % page
    return dict(pages=pages, kv=kv, new=new, table=table, begin=begin, seq=seq, pos=pos, slot=slot)


def _quantised(x, gs):
    """Codes and scales of x [..., D] in groups of gs values: scale = absmax / 7 (1 where that is below 1e-8), codes
    x / scale rounded half away from zero, every step in 32 bits."""
    t = x.reshape(*x.shape[:-1], -1, gs)
    # a tensor divisor: torch multiplies by the reciprocal of a scalar one
    s = t.abs().amax(-1, keepdim=True) / torch.full((), 7.0, device=x.device).expand(1)
    s = torch.where(s < 1e-8, torch.ones_like(s), s)
    d = t / s
    r = d.abs().floor()
    code = (d.sign() * (r + (d.abs() - r >= 0.5))).clamp(-8, 7)
    return code, s


def _packed(code):
    """Bytes of integer codes [..., D]: the even value in the low nibble."""
    q = code.to(torch.int32) & 15
    return (q[..., 0::2] | (q[..., 1::2] << 4)).to(torch.uint8)


def _values(byte):
    """Integer codes (float) of packed bytes, the last dimension twice as long."""
    b = byte.to(torch.int32)
    q = torch.stack([b & 15, b >> 4], -1).reshape(*b.shape[:-1], -1)
    return (q - 16 * (q >= 8)).float()


def _cache(c, seed, pages):
    """One layer's pages full of quantised N(0, 1) keys and values."""
    g, Hk, D, gs, page = _gen(seed, 1), c["Hk"], c["D"], c["gs"], c["page"]

    def half():
        code, s = _quantised(_normal(g, pages, Hk, page, D), gs)
        return _packed(code.reshape(pages, Hk, page, D)), s.reshape(pages, Hk, page, D // gs).contiguous()

    k, ks = half()
    v, vs = half()
    v = v.reshape(pages, Hk, page // 16, 16, 16, D // 32).transpose(3, 4).contiguous()
    return k.reshape(-1), v.reshape(-1), ks.reshape(-1), vs.reshape(-1)


def _rope(n, D):
    """(cos, sin) of position times frequency: [n][D/2][2]."""
    freq = 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    a = torch.arange(n, dtype=torch.float64)[:, None] * freq
    return torch.stack([a.cos(), a.sin()], -1).float().cuda().contiguous()


def _tree(r, new):
    """Ancestor bits of every row: row i of a sequence hangs below a row of the first half of those before it, or below the cached prefix."""
    bits = []
    for n in new:
        of = []
        for i in range(int(n)):
            up = -1 if i == 0 else int(r.randint(-1, (i + 1) // 2))
            of.append((1 << i) | (of[up] if up >= 0 else 0))
        bits += of
    return torch.from_numpy(np.array(bits, dtype=np.uint64).view(np.int64)).cuda()


def prepare(case, seed):
    c = case
    s = {"case": c}
    if c["kind"] == "tables":
        keep, new = _lengths(c)
        r, page = np.random.RandomState(seed % (1 << 31)), c["page"]
        # before the rollback each sequence had up to rows - 1 rejected rows more
        old = keep + (np.arange(c["B"]) * 7 % c["rows"] if c["rollback"] else 0)
        held = _pages_of(old, page)
        width = int(_pages_of(np.maximum(old, keep + new), page).max())
        pages = int(held.sum() + _pages_of(new, page).sum() + c["B"] + 7)
        order = r.permutation(pages)
        table = np.full((c["B"], width), -1, np.int64)
        table[np.arange(width) < held[:, None]] = order[:held.sum()]
        free = np.full(pages, -1, np.int64)
        free[:pages - held.sum()] = order[held.sum():]
        T = int(new.sum())
        s.update(old=_i32(old), keep=_i32(keep), new=_i32(new), table=_i32(table), free=_i32(free),
                 count=_i32([pages - held.sum()]), pages=pages, T=T, next=torch.empty_like(_i32(table)))
        s.update({k: torch.full((n,), -7, dtype=torch.int32, device="cuda") for k, n in
                  (("left", 1), ("begin", c["B"] + 1), ("seq", T), ("pos", T), ("slot", T),
                   ("kv", c["B"]), ("status", 4))})
        return s
    if c["kind"] == "logprobs":
        g = _gen(seed)
        rows, V = c["rows"], c["V"]
        # flat rows and peaked ones
        x = _normal(g, rows, V) * (1.0 + 3.0 * torch.rand(rows, 1, generator=g, device="cuda"))
        if c["masked"]:                                # tokens that a grammar rules out
            x = torch.where(torch.rand(rows, V, generator=g, device="cuda") < 0.3, -math.inf, x)
        tok = (x - torch.empty_like(x).exponential_(generator=g).log()).argmax(-1).int()
        f, i = dict(device="cuda"), dict(dtype=torch.int32, device="cuda")
        s.update(x=x.contiguous(), tok=tok, lp=torch.zeros(rows, **f), rank=torch.zeros(rows, **i),
                 entropy=torch.zeros(rows, **f), top=torch.zeros(rows, c["top"], **i),
                 top_lp=torch.zeros(rows, c["top"], **f), ws=torch.empty(32 << 20, dtype=torch.uint8, **f))
        return s
    b = _batch(c, seed)
    H, Hk, D, T = c["H"], c["Hk"], c["D"], len(b["seq"])
    g = _gen(seed)
    s.update({k: _i32(b[k]) for k in ("table", "begin", "seq", "pos", "slot", "kv", "new")},
             pages=b["pages"], T=T, most=int(b["new"].max()), longest=int(b["kv"].max()),
             status=torch.zeros(4, dtype=torch.int32, device="cuda"))
    if c["kind"] == "append":
        n, groups = b["pages"] * c["page"] * Hk * D // 2, b["pages"] * c["page"] * Hk * (D // c["gs"])
        s["qkv"] = _normal(g, T, (H + 2 * Hk) * D)
        s["rope"] = _rope(s["longest"], D)
        s["pool"] = (torch.zeros(n, dtype=torch.uint8, device="cuda"),
                     torch.zeros(n, dtype=torch.uint8, device="cuda"),
                     torch.zeros(groups, device="cuda"), torch.zeros(groups, device="cuda"))
        s["q"] = torch.zeros(T, H, D, device="cuda")
        s["k"], s["v"] = torch.zeros(T, Hk, D, device="cuda"), torch.zeros(T, Hk, D, device="cuda")
        return s
    s["pool"] = _cache(c, seed, b["pages"])
    s["q"] = _normal(g, T, H, D)
    s["o"] = torch.zeros(T, H, D, device="cuda")
    s["lse"] = torch.zeros(T, H, device="cuda") if c["lse"] else None
    s["anc"] = _tree(np.random.RandomState(seed % (1 << 31) ^ 77), b["new"]) if c["tree"] else None
    s["ws"] = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------- the plain forms

def _plain_tables(s):
    c = s["case"]
    page, table, keep, new, count = c["page"], s["table"], s["keep"], s["new"], s["count"]
    at = torch.arange(table.shape[1], device="cuda")
    kv = keep + new
    held, need = (s["old"] + page - 1) // page, (kv + page - 1) // page
    # the pages given back, sequence by sequence, on top of the stack
    back = ((at >= need[:, None]) & (at < held[:, None])).flatten()
    given = back.sum()
    stack = torch.cat([s["free"], s["free"].new_zeros(1)])
    spare = s["free"].numel()
    stack[torch.where(back, count + torch.cumsum(back, 0) - 1, spare)] = table.flatten()
    count = count + given
    # then the pages taken, from the top down
    take = (need - held).clamp(min=0)
    before = torch.cumsum(take, 0) - take
    new_page = (at >= held[:, None]) & (at < need[:, None])
    src = torch.where(new_page, count - 1 - before[:, None] - (at - held[:, None]), 0)
    table = torch.where(at < need[:, None], torch.where(new_page, stack[src], table), -1)
    begin = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    t = torch.arange(s["T"], device="cuda")
    seq = torch.searchsorted(begin, t, right=True) - 1
    pos = t - begin[seq] + keep[seq]
    slot = table[seq, pos // page] * page + pos % page
    left = count - take.sum()
    # the stack's entries below the old count stay, those above the new one too
    at = torch.arange(spare, device="cuda")
    free = torch.where((at >= s["count"]) & (at < left), stack[:-1], s["free"])
    return {"table": table.int(), "begin": begin.int(),
            "seq": seq.int(), "pos": pos.int(), "slot": slot.int(), "kv": kv.int(), "left": left.int(),
            "free": free.int()}


def _plain_append(s):
    c = s["case"]
    H, Hk, D, gs = c["H"], c["Hk"], c["D"], c["gs"]
    x = s["qkv"].reshape(s["T"], H + 2 * Hk, D)
    cs = s["rope"][s["pos"].long()][:, None]
    co, si = cs[..., 0], cs[..., 1]
    x0, x1 = x[:, :H + Hk, :D // 2], x[:, :H + Hk, D // 2:]
    turned = torch.cat([x0 * co - x1 * si, x0 * si + x1 * co], -1)
    back = lambda y: (lambda q: (q[0] * q[1]).reshape(y.shape))(_quantised(y, gs))  # noqa: E731
    return {"q": turned[:, :H], "k": back(turned[:, H:]), "v": back(x[:, H + Hk:])}


def _dequantised(s):
    """Keys and values of every page: [pages, Hk, page, D]."""
    c = s["case"]
    Hk, D, gs, page, n = c["Hk"], c["D"], c["gs"], c["page"], s["pages"]
    k, v, ks, vs = s["pool"]
    v = v.reshape(n, Hk, page // 16, 16, 16, D // 32).transpose(3, 4)
    wide = lambda q, x: (_values(q.reshape(n, Hk, page, D // 2)).reshape(n, Hk, page, D // gs, gs) *  # noqa: E731
                         x.reshape(n, Hk, page, D // gs, 1)).reshape(n, Hk, page, D)
    return wide(k, ks), wide(v, vs)


def _plain_attention(s):
    """Every sequence padded to the longest one and to the most rows."""
    c = s["case"]
    H, Hk, D, B, page = c["H"], c["Hk"], c["D"], c["B"], c["page"]
    n, m = s["most"], s["longest"]
    k, v = _dequantised(s)
    tab = torch.where(s["table"] >= 0, s["table"], 0).long()
    # [B, Hk, keys, D] of each sequence's pages
    kk = k[tab].transpose(1, 2).reshape(B, Hk, -1, D)[:, :, :m]
    vv = v[tab].transpose(1, 2).reshape(B, Hk, -1, D)[:, :, :m]
    seq = s["seq"].long()
    i = torch.arange(s["T"], device="cuda") - s["begin"][seq]
    q = torch.zeros(B, n, H, D, device="cuda")
    q[seq, i] = s["q"]
    G = H // Hk
    q = q.reshape(B, n, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * n, D)
    sc = torch.matmul(q, kk.transpose(2, 3).contiguous()).reshape(B, Hk, G, n, m) * (1.0 / math.sqrt(D))
    j = torch.arange(m, device="cuda")
    base = (s["kv"] - s["new"])[:, None, None]
    if c["tree"]:
        anc = torch.zeros(B, n, dtype=torch.int64, device="cuda")
        anc[seq, i] = s["anc"]
        d = (j - base).clamp(0, 63)
        see = (j < base) | ((((anc[:, :, None] >> d) & 1) > 0) & (j < s["kv"][:, None, None]))
    else:
        see = j <= base + torch.arange(n, device="cuda")[None, :, None]
    sc = torch.where(see[:, None, None], sc, -math.inf)
    top = sc.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    e = torch.exp(sc - top)
    z = e.sum(-1, keepdim=True)
    o = torch.matmul(e.reshape(B, Hk, G * n, m), vv).reshape(B, Hk, G, n, D)
    o = torch.where(z > 0, o / z, 0.0).permute(0, 3, 1, 2, 4).reshape(B, n, H, D)[seq, i]
    if not c["lse"]:
        return {"o": o}
    lse = (top + z.log()).reshape(B, H, n).transpose(1, 2)[seq, i]
    return {"o": o, "lse": lse}


def _plain_logprobs(s):
    x, tok = s["x"], s["tok"].long()[:, None]
    top = x.amax(1, keepdim=True)
    d = x - top
    e = torch.exp(d)
    z = e.sum(1, keepdim=True)
    logz = z.log()
    given = x.gather(1, tok)
    at = torch.arange(x.shape[1], device="cuda")
    rank = ((x > given) | ((x == given) & (at < tok))).sum(1)
    entropy = logz[:, 0] - torch.where(e > 0, e * d, 0.0).sum(1) / z[:, 0]
    best, order = torch.sort(x, dim=1, descending=True, stable=True)
    n = min(s["case"]["top"], x.shape[1])
    return {"lp": (given - top - logz)[:, 0], "rank": rank.int(), "entropy": entropy,
            "top": order[:, :n].int(), "top_lp": best[:, :n] - top - logz}


# ----------------------------------------------------- the library's calls

def _own_call(s):
    """The calls of a pass, their arguments bound once, as a program that keeps its batch would."""
    import ctypes as C

    import cogito_amd
    from cogito_amd.capi import CgxKvPagedInt4, CgxPagedStep, last_error
    lib = cogito_amd.load()
    c = s["case"]

    def ok(rc):
        if rc:
            raise RuntimeError(last_error(lib))

    ok(lib.cgx_init(0))
    p = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
    if c["kind"] == "logprobs":
        n = min(c["top"], c["V"])
        args = (p(s["x"]), c["V"], c["rows"], c["V"], p(s["tok"]), n, p(s["lp"]), p(s["rank"]),
                p(s["entropy"]), p(s["top"]) if n else None, p(s["top_lp"]) if n else None,
                p(s["ws"]), s["ws"].numel())
        out = {k: s[k] for k in ("lp", "rank", "entropy")}
        out.update(top=s["top"][:, :n], top_lp=s["top_lp"][:, :n])

        def call():
            ok(lib.cgx_token_logprobs_dev(*args))
            return out
        return call
    step = CgxPagedStep(seqs=c["B"], rows=s["T"], max_rows=0, table_ld=s["table"].shape[1])
    step.table, step.row_begin, step.row_seq = p(s["table"]), p(s["begin"]), p(s["seq"])
    step.row_pos, step.row_slot, step.kv_len = p(s["pos"]), p(s["slot"]), p(s["kv"])
    step.status = p(s["status"])
    if c["kind"] == "tables":
        step.kv_old, step.kv_keep, step.rows_new = p(s["old"]), p(s["keep"]), p(s["new"])
        step.table_old, step.table = p(s["table"]), p(s["next"])
        args = (C.byref(step), c["page"], s["pages"], p(s["free"]), p(s["count"]), p(s["left"]))
        out = {k: s[k] for k in ("begin", "seq", "pos", "slot", "kv", "left", "free")}
        out["table"] = s["next"]

        def call(step=step):
            ok(lib.cgx_paged_plan_dev(*args))
            return out
        return call
    cache = CgxKvPagedInt4(num_layers=1, num_pages=s["pages"], page_size=c["page"], n_heads=c["Hk"],
                           head_dim=c["D"], group_size=c["gs"])
    cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales = map(p, s["pool"])
    step.max_rows = s["most"]
    if c["kind"] == "append":
        put = (C.byref(cache), 0, C.byref(step), p(s["qkv"]), s["qkv"].shape[1], c["H"], p(s["rope"]),
               s["longest"], p(s["q"]))
        get = (C.byref(cache), 0, p(s["slot"]), s["T"], p(s["k"]), p(s["v"]))
        out = {k: s[k] for k in ("q", "k", "v")}

        def call(cache=cache, step=step):
            ok(lib.cgx_kv_paged_append_dev(*put))
            ok(lib.cgx_kv_paged_gather_dev(*get))
            return out
        return call
    args = (C.byref(cache), 0, C.byref(step), p(s["q"]), c["H"], p(s["anc"]), None, p(s["o"]), p(s["lse"]),
            p(s["ws"]), s["ws"].numel())
    out = {"o": s["o"], "lse": s["lse"]} if c["lse"] else {"o": s["o"]}

    def call(cache=cache, step=step):
        ok(lib.cgx_attention_paged_dev(*args))
        return out
    return call


def run(state):
    s = state
    if own:
        if "call" not in s:
            s["call"] = _own_call(s)
        return s["call"]()
    return {"tables": _plain_tables, "append": _plain_append, "attention": _plain_attention,
            "logprobs": _plain_logprobs}[s["case"]["kind"]](s)


# ----------------------------------------------------------- work, 64 bits

def work(case):
    c = case
    if c["kind"] == "logprobs":
        return {"bytes": 4 * c["rows"] * (c["V"] + 4 + 2 * c["top"]), "flops": 0}
    old, new = _lengths(c)
    T, page = int(new.sum()), c["page"]
    taken = int((_pages_of(old + new, page) - _pages_of(old, page)).sum())
    if c["kind"] == "tables":
        return {"bytes": 4 * (4 * c["B"] + 2 * taken + 3 * T), "flops": 0}
    H, Hk, D, gs = c["H"], c["Hk"], c["D"], c["gs"]
    packed = Hk * (D // 2 + 4 * D // gs)
    if c["kind"] == "append":
        # rows in, rotated queries and packed rows out, packed rows in, values out
        return {"bytes": T * (4 * (H + 2 * Hk) * D + 4 * H * D + 4 * packed + 8 * Hk * D), "flops": 0}
    seen = int((new * old + new * (new + 1) // 2).sum())
    return {"bytes": int((old + new).sum()) * 2 * packed + 8 * T * H * D, "flops": 4 * seen * H * D}


def exact(case, seed):
    c = case
    if c["kind"] == "tables":
        return None                                    # whole numbers only
    s = prepare(c, seed)
    if c["kind"] == "logprobs":
        x = s["x"].double()
        lse = torch.logsumexp(x, 1)
        lp = x - lse[:, None]
        n = min(c["top"], c["V"])
        return {"lp": lp[torch.arange(len(x)), s["tok"].long()], "rank": None,
                "entropy": -torch.nan_to_num(lp.exp() * lp, nan=0.0).sum(1), "top": None,
                "top_lp": torch.topk(lp, n, 1).values}
    H, Hk, D, gs, page = c["H"], c["Hk"], c["D"], c["gs"], c["page"]
    if c["kind"] == "append":
        # keys are rotated, and both quantised, in 32 bits by definition
        x = s["qkv"].cpu().numpy().reshape(-1, H + 2 * Hk, D)
        cs = s["rope"].cpu().numpy()[s["pos"].cpu().numpy()][:, None]

        def turn(y, kind):
            y, a = y.astype(kind), cs.astype(kind)
            lo, hi = y[..., :D // 2], y[..., D // 2:]
            return np.concatenate([lo * a[..., 0] - hi * a[..., 1], lo * a[..., 1] + hi * a[..., 0]], -1)

        def stored(y):
            t = y.reshape(len(y), Hk, D // gs, gs)
            sc = np.abs(t).max(-1, keepdims=True) / np.float32(7)
            sc = np.where(sc < np.float32(1e-8), np.float32(1), sc)
            r = (t / sc).astype(np.float64)
            code = np.clip(np.sign(r) * np.floor(np.abs(r) + 0.5), -8, 7)
            return (code * sc.astype(np.float64)).reshape(y.shape)

        return {"q": turn(x[:, :H], np.float64), "k": stored(turn(x[:, H:H + Hk], np.float32)),
                "v": stored(np.ascontiguousarray(x[:, H + Hk:]))}
    k8, v8, ks, vs = s["pool"]
    k8 = k8.view(s["pages"], Hk, page, D // 2)
    v8 = v8.view(s["pages"], Hk, page // 16, 16, 16, D // 32)
    ks, vs = ks.view(s["pages"], Hk, page, D // gs), vs.view(s["pages"], Hk, page, D // gs)
    code = torch.tensor([n if n < 8 else n - 16 for n in range(16)], dtype=torch.float64, device="cuda")
    out, lses, G = [], [], H // Hk
    begin, kv = s["begin"].tolist(), s["kv"].tolist()
    for b in range(c["B"]):
        L, r0, r1 = kv[b], begin[b], begin[b + 1]
        tab = s["table"][b, :_pages_of(L, page)].long()
        os, ls = [], []
        for h in range(Hk):
            def wide(byte, sc):
                y = code[torch.stack([byte & 15, byte >> 4], -1).long()].reshape(-1, D // gs, gs)
                return (y * sc.reshape(-1, D // gs, 1).double()).reshape(-1, D)[:L]
            K = wide(k8[tab, h], ks[tab, h])
            V = wide(v8[tab, h].transpose(2, 3).contiguous(), vs[tab, h])
            q = s["q"][r0:r1, h * G:(h + 1) * G].double().reshape(-1, D)
            z = (q @ K.T / math.sqrt(D)).reshape(r1 - r0, G, L)
            at, base = torch.arange(L, device="cuda"), L - (r1 - r0)
            if c["tree"]:
                bit = (s["anc"][r0:r1, None] >> (at - base).clamp(min=0)) & 1
                hide = (at >= base) & (bit == 0)
            else:
                hide = at > base + torch.arange(r1 - r0, device="cuda")[:, None]
            z = z.masked_fill(hide[:, None], -math.inf)
            ls.append(torch.logsumexp(z, -1))
            os.append((torch.softmax(z, -1).reshape(-1, L) @ V).reshape(r1 - r0, G, D))
        out.append(torch.cat(os, 1))
        lses.append(torch.cat(ls, 1))
    o = {"o": torch.cat(out)}
    return dict(o, lse=torch.cat(lses)) if c["lse"] else o
