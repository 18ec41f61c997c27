"""Microscaled 4-bit weights and the loss over a vocabulary of them, in plain form and as the library's calls.

  quantize  rows to blocks of 32 values with one power of two each, 4-bit (E2M1) or 6-bit (E2M3)
            elements, and read back (cgx_mx_quantize_dev, cgx_mx_dequantize_dev)
  matmul    rows times a 4-bit weight; the rows as they are or quantised like the weight
            (cgx_matmul_mx_dev)
  loss      cross entropy of each row's target over the vocabulary of an lm_head, from the hidden
            rows (cgx_token_loss_mx_dev)
  train     the same with its gradient with respect to the hidden rows
            (cgx_token_loss_mx_grad_dev)

A block's scale is 2^E, E = floor(log2 of its largest magnitude) - 2, at least -126, stored as E + 127;
elements are rounded to the nearest, ties to even, and saturate at 6 (E2M1) or 7.5 (E2M3). Weights are
held as [outputs][inputs]: two codes a byte, the even one in its low nibble, and one scale a block.

Sizes are those of the benchmark's stacks (d 4096 and 768, gate|up of 22016 outputs, down of 11008
inputs, vocabularies of 32000, 50257 and 128256, gamma 4) and prompts up to 2048; `draw` spreads over the
ranges around them.
"""
from __future__ import annotations

import math

import torch

own = False


# ------------------------------------------------------------------ cases

def _quantize(rows, cols, fmt, **name):
    return dict(name, kind="quantize", rows=rows, cols=cols, fmt=fmt)


def _matmul(M, K, N, act, **name):
    return dict(name, kind="matmul", M=M, K=K, N=N, act=act)


def _loss(rows, K, V, act, **name):
    return dict(name, kind="loss", rows=rows, K=K, V=V, act=act)


def _train(rows, K, V, act, **name):
    return dict(name, kind="train", rows=rows, K=K, V=V, act=act)


def listed():
    return [
        # the hidden rows of one verified chain (gamma 4): latency
        _quantize(5, 4096, "fp4", name="quantize_rows"),
        # a down projection's weight, read in once
        _quantize(11008, 4096, "fp4", name="quantize_weight"),
        # a prompt's activations, a last block of 8 values
        _quantize(2039, 1000, "fp6", name="quantize_prompt"),
        # one decoded token through gate|up: the weight's bytes
        _matmul(1, 4096, 22016, "fp32", name="matmul_decode"),
        # a verified chain through the O projection: latency
        _matmul(5, 4096, 4096, "fp32", name="matmul_verify"),
        # eight verified chains through the down projection
        _matmul(40, 11008, 4096, "fp32", name="matmul_batch"),
        # a prompt of odd length, sizes that end inside a tile, 6-bit rows
        _matmul(301, 1000, 2401, "fp6", name="matmul_ragged"),
        # a long prompt through gate|up, both sides in 4 bits: the matrix cores
        _matmul(2039, 4096, 22016, "fp4", name="matmul_prompt"),
        # emitted tokens of one chain scored by the small decoder: latency
        _loss(5, 768, 32000, "fp32", name="loss_verify"),
        # a scored prompt over the large vocabulary
        _loss(301, 4096, 128256, "fp32", name="loss_prompt"),
        # a short sequence of the small decoder's draft head
        _train(61, 768, 50257, "fp32", name="train_small"),
        # a training batch of a draft head over the target's lm_head
        _train(1024, 4096, 32000, "fp32", name="train_draft"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "matmul", "matmul", "loss", "train"])
    act = rng.choice(["fp32", "fp32", "fp4", "fp6"])
    if kind == "quantize":
        rows, cols = _log_int(rng, 1, 11008), rng.choice([4096, _log_int(rng, 1, 11008), _log_int(rng, 1, 11008)])
        while rows > 1 and rows * cols > 11008 * 4096:
            rows //= 2
        return _quantize(rows, cols, rng.choice(["fp4", "fp6"]))
    if kind == "matmul":
        M = rng.choice([1, _log_int(rng, 1, 16), _log_int(rng, 1, 64), _log_int(rng, 1, 2048)])
        K, N = rng.choice([(4096, _log_int(rng, 16, 22016)), (768, _log_int(rng, 16, 22016)),
                           (_log_int(rng, 32, 11008), 4096), (_log_int(rng, 32, 11008), 6144),
                           (_log_int(rng, 32, 11008), _log_int(rng, 16, 22016))])
        while M > 1 and M * K * N > 2039 * 4096 * 22016:
            M //= 2
        return _matmul(M, K, N, act)
    rows = rng.choice([_log_int(rng, 1, 16), _log_int(rng, 1, 2048), _log_int(rng, 64, 2048)])
    K, V = rng.choice([(4096, _log_int(rng, 100, 128256)), (768, _log_int(rng, 100, 128256)),
                       (_log_int(rng, 32, 4096), 32000), (_log_int(rng, 32, 4096), 128256),
                       (_log_int(rng, 32, 4096), 50257)])
    most = 1024 * 4096 * 32000 if kind == "loss" else 1024 * 4096 * 16000
    while rows > 1 and rows * K * V > most:
        rows //= 2
    return (_loss if kind == "loss" else _train)(rows, K, V, act)


# ----------------------------------------------------------------- inputs

def _gen(seed, salt=0):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + salt)


def _rows(g, n, K):
    """Hidden rows: channels of different size, rows of different size."""
    x = torch.randn(n, K, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(K, generator=g, device="cuda"))
    return x * torch.exp(0.3 * torch.randn(n, 1, generator=g, device="cuda"))


def _weight(g, N, K, size):
    """Codes [N][ceil(K/32) * 16] and scales [N][ceil(K/32)] of a normal weight, some rows ten times smaller."""
    codes, scales = [], []
    for n in range(0, N, 8192):
        w = torch.randn(min(8192, N - n), K, generator=g, device="cuda") * size
        w *= torch.where(torch.rand(len(w), 1, generator=g, device="cuda") < 0.02, 0.1, 1.0)
        v, s = _blocks(w, "fp4")
        c = (_CODE(v) | torch.where(torch.signbit(v), 8, 0)).reshape(len(w), -1)
        codes.append((c[:, 0::2] | (c[:, 1::2] << 4)).to(torch.uint8))
        scales.append(s.to(torch.uint8))
    return torch.cat(codes), torch.cat(scales)


def _CODE(v):
    a = v.abs()
    return torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.int32)


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": c}
    if c["kind"] == "quantize":
        rows, cols = c["rows"], c["cols"]
        n = -(-cols // 32)
        s["x"] = _rows(g, rows, cols)
        s["codes"] = torch.zeros(rows, n * (16 if c["fmt"] == "fp4" else 24), dtype=torch.uint8, device="cuda")
        s["scales"] = torch.zeros(rows, n, dtype=torch.uint8, device="cuda")
        s["y"] = torch.zeros(rows, cols, device="cuda")
        return s
    K, N, M = c["K"], c.get("N", c.get("V")), c.get("M", c.get("rows"))
    s["x"] = _rows(g, M, K)
    # products and logits of size 1 to 3
    s["codes"], s["scales"] = _weight(g, N, K, 1.5 / math.sqrt(K))
    if c["kind"] == "matmul":
        s["y"] = torch.zeros(M, N, device="cuda")
        return s
    # half the targets likely ones, a tenth of a larger batch's padding
    t = torch.randint(0, N, (M,), generator=g, device="cuda")
    z = s["x"][:64] @ _values(s["codes"][:4096], s["scales"][:4096], K).T
    t[:64:2] = z.argmax(1)[::2]
    if M > 16:
        t = torch.where(torch.rand(M, generator=g, device="cuda") < 0.1, -1, t)
    s["targets"] = t.int()
    s["loss"], s["lse"] = torch.zeros(M, device="cuda"), torch.zeros(M, device="cuda")
    if c["kind"] == "train":
        s["dloss"] = torch.full((M,), 1.0 / max(1, int((t >= 0).sum())), device="cuda")
        s["dh"] = torch.zeros(M, K, device="cuda")
    return s


# ------------------------------------------------------- the plain forms

def _power(byte):
    """2^(byte - 127), for bytes from 1 to 254."""
    return (byte.to(torch.int32) << 23).view(torch.float32)


def _blocks(x, fmt):
    """x [..., K] in blocks of 32, the last one filled up with zeros: rounded values of each block over its scale
    [..., blocks, 32], and scale bytes [..., blocks]."""
    K = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, -K % 32)).reshape(*x.shape[:-1], -1, 32)
    top = x.abs().amax(-1)
    byte = ((top.view(torch.int32) >> 23) - 2).clamp(min=1)
    v = x * _power(254 - byte)[..., None]
    a = v.abs()
    if fmt == "fp4":
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
        a = (torch.round(a / step) * step).clamp(max=6.0)
    else:
        step = torch.where(a < 2, 0.125, torch.where(a < 4, 0.25, 0.5))
        a = (torch.round(a / step) * step).clamp(max=7.5)
    return torch.copysign(a, v), byte


def _rounded(x, fmt):
    """x as its quantised values."""
    v, byte = _blocks(x, fmt)
    return (v * _power(byte)[..., None]).flatten(-2)[..., :x.shape[-1]]


def _values(codes, scales, K):
    """Values [N][K] of a weight's codes."""
    b = codes.to(torch.int32)
    q = torch.stack([b & 15, b >> 4], -1).reshape(len(b), -1, 32)
    m = q & 7
    v = torch.where(m < 4, m * 0.5, torch.where(m < 6, m - 2.0, m * 2.0 - 8.0))
    v = torch.where(q > 7, -v, v) * _power(scales)[..., None]
    return v.flatten(1)[:, :K]


def _plain(s):
    c = s["case"]
    if c["kind"] == "quantize":
        return {"y": _rounded(s["x"], c["fmt"])}
    x = s["x"] if c["act"] == "fp32" else _rounded(s["x"], c["act"])
    w = _values(s["codes"], s["scales"], c["K"])
    z = x @ w.T
    if c["kind"] == "matmul":
        return {"y": z}
    top = z.amax(1)
    e = torch.exp(z - top[:, None])
    total = e.sum(1)
    lse = top + total.log()
    t = s["targets"].long()
    taken = t >= 0
    at = torch.where(taken, t, 0)[:, None]
    out = {"loss": torch.where(taken, lse - z.gather(1, at)[:, 0], 0.0), "lse": lse}
    if c["kind"] == "loss":
        return out
    e /= total[:, None]
    e.scatter_add_(1, at, -torch.ones_like(at, dtype=e.dtype))
    out["dh"] = (e @ w) * torch.where(taken, s["dloss"], 0.0)[:, None]
    return out


# ----------------------------------------------------- the library's calls

class _Handle:
    """A weight laid out for the library, as a program keeps it."""

    def __init__(self, lib, s, K, N, grad):
        self.lib = lib
        torch.cuda.current_stream().synchronize()     # the codes are made on torch's stream
        self.ptr = lib.cgx_mx_weight_new(s["codes"].data_ptr(), s["scales"].data_ptr(), K, N, grad)

    def __del__(self):
        if self.ptr:
            self.lib.cgx_mx_weight_free(self.ptr)


def _own_call(s):
    """The calls of a pass, their arguments bound once, as a program that keeps its weight would."""
    import cogito_amd
    from cogito_amd.capi import CGX_MX_FP4, CGX_MX_FP6, CGX_MX_FP32, last_error
    lib = cogito_amd.load()
    c = s["case"]

    def ok(rc):
        if rc:
            raise RuntimeError(last_error(lib))

    ok(lib.cgx_init(0))
    form = {"fp4": CGX_MX_FP4, "fp6": CGX_MX_FP6, "fp32": CGX_MX_FP32}
    p = lambda t: t.data_ptr()  # noqa: E731
    if c["kind"] == "quantize":
        rows, cols, f = c["rows"], c["cols"], form[c["fmt"]]
        put = (p(s["x"]), cols, rows, cols, f, p(s["codes"]), p(s["scales"]))
        get = (p(s["codes"]), p(s["scales"]), rows, cols, f, p(s["y"]), cols)

        def call():
            ok(lib.cgx_mx_quantize_dev(*put))
            ok(lib.cgx_mx_dequantize_dev(*get))
            return {"y": s["y"]}
        return call
    K, N, M = c["K"], c.get("N", c.get("V")), c.get("M", c.get("rows"))
    act, train = form[c["act"]], c["kind"] == "train"
    w = s["handle"] = _Handle(lib, s, K, N, 1 if train else 0)
    if not w.ptr:
        raise RuntimeError(last_error(lib))
    if c["kind"] == "matmul":
        n = lib.cgx_matmul_mx_ws(w.ptr, M, act)
        s["ws"] = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
        args = (p(s["x"]), K, M, w.ptr, act, p(s["y"]), N, p(s["ws"]), n)

        def call():
            ok(lib.cgx_matmul_mx_dev(*args))
            return {"y": s["y"]}
        return call
    n = lib.cgx_token_loss_mx_ws(w.ptr, M, act, 1 if train else 0)
    s["ws"] = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
    fwd = (p(s["x"]), K, M, w.ptr, act, p(s["targets"]), p(s["loss"]), p(s["lse"]), p(s["ws"]), n)
    out = {"loss": s["loss"], "lse": s["lse"]}
    if not train:
        def call():
            ok(lib.cgx_token_loss_mx_dev(*fwd))
            return out
        return call
    bwd = (p(s["x"]), K, M, w.ptr, act, p(s["targets"]), p(s["lse"]), p(s["dloss"]), p(s["dh"]), K, p(s["ws"]), n)
    out["dh"] = s["dh"]

    def call():
        ok(lib.cgx_token_loss_mx_dev(*fwd))
        ok(lib.cgx_token_loss_mx_grad_dev(*bwd))
        return out
    return call


def run(state):
    s = state
    if own:
        if "call" not in s:
            s["call"] = _own_call(s)
        return s["call"]()
    return _plain(s)


# ----------------------------------------------------------- work, 64 bits

def work(case):
    c = case
    if c["kind"] == "quantize":
        n, blocks = c["rows"] * c["cols"], c["rows"] * -(-c["cols"] // 32)
        # values in, codes and scales out and in again, values out
        return {"bytes": 8 * n + 2 * blocks * (17 if c["fmt"] == "fp4" else 25), "flops": 0}
    K, N, M = c["K"], c.get("N", c.get("V")), c.get("M", c.get("rows"))
    weight = N * -(-K // 32) * 17
    if c["kind"] == "matmul":
        return {"bytes": weight + 4 * M * (K + N), "flops": 2 * M * N * K}
    if c["kind"] == "loss":
        return {"bytes": weight + 4 * M * (K + 3), "flops": 2 * M * N * K}
    return {"bytes": weight + 4 * M * (2 * K + 4), "flops": 4 * M * N * K}


def _read_back(x, fmt):
    """The nearest element of every value, by search in a table of them, in 64 bits."""
    man = 1 if fmt == "fp4" else 3
    table = [m / (1 << man) for m in range(1 << man)]
    table += [(1 + m / (1 << man)) * 2.0 ** e for e in range(3) for m in range(1 << man)]
    table = torch.tensor(table, dtype=torch.float64, device="cuda")
    if x.shape[1] % 32:
        x = torch.cat([x, x.new_zeros(len(x), 32 - x.shape[1] % 32)], 1)
    t = x.reshape(len(x), -1, 32)
    e = torch.frexp(t.abs().max(2, keepdim=True).values).exponent.double() - 3
    scale = torch.pow(2.0, torch.clamp(e, min=-126.0))
    a = t.abs() / scale
    up = torch.searchsorted(table, a).clamp(max=len(table) - 1)
    lo = (up - 1).clamp(min=0)
    over, under = table[up] - a, a - table[lo]
    # the nearer one, of two as near the one whose last bit is 0
    at = torch.where((over < under) | ((over == under) & (up % 2 == 0)) | (a >= table[-1]), up, lo)
    return torch.sign(t) * table[at] * scale


def exact(case, seed):
    c, s = case, prepare(case, seed)
    x = s["x"].double()
    if c["kind"] == "quantize":
        y = [_read_back(r, c["fmt"]).reshape(len(r), -1)[:, :c["cols"]] for r in x.split(2048)]
        return {"y": torch.cat(y)}
    K = c["K"]
    if c["act"] != "fp32":
        x = _read_back(x, c["act"]).reshape(len(x), -1)[:, :K]
    lut = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device="cuda")

    def part(n):
        """Rows n .. n + 16383 of the weight."""
        b = s["codes"][n:n + 16384].long()
        w = torch.empty(*b.shape, 2, dtype=torch.float64, device="cuda")
        w[..., 0], w[..., 1] = lut[b % 16], lut[b // 16]
        w = w.reshape(len(b), -1, 32) * torch.pow(2.0, s["scales"][n:n + 16384].double() - 127)[:, :, None]
        return w.reshape(len(b), -1)[:, :K]

    N = c.get("N", c.get("V"))
    z = torch.cat([x @ part(n).T for n in range(0, N, 16384)], 1)
    if c["kind"] == "matmul":
        return {"y": z}
    lse = torch.logsumexp(z, 1)
    t = s["targets"].long()
    row = torch.arange(len(z), device="cuda")
    out = {"lse": lse, "loss": (lse - z[row, t.clamp(min=0)]).masked_fill(t < 0, 0)}
    if c["kind"] == "loss":
        return out
    p = torch.softmax(z, 1)
    p[row, t.clamp(min=0)] -= 1
    p *= s["dloss"].double().masked_fill(t < 0, 0)[:, None]
    out["dh"] = sum(p[:, n:n + 16384] @ part(n) for n in range(0, N, 16384))
    return out
