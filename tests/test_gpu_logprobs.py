"""GPU: token log probabilities, ranks, entropies and top alternatives against 64 bits.

Tolerances: an exponential's argument d = x - max, |d| up to R (the row's
range), is rounded once or twice (2 R 2^-24 relative in the term), sums of
the terms add a few roundings of their own (at most log2 of the count, 17, in
tree order): with R <= 40 that is 100 * 2^-24 = 6e-6 relative in z, and as much
absolute in log z.  A term's weight falls with |d| as its error grows, so the
sums are nearer than that; log probabilities are held to 6e-6 + 2^-23 |lp| and
entropies, whose second sum has the weights d, to 6e-6 (1 + H)."""
from __future__ import annotations

import numpy as np
import pytest

from cogito_amd.capi import DeviceArray, last_error

pytestmark = pytest.mark.gpu


def _run(lib, x, tok, n_top, ld=None, want=("lp", "rank", "ent")):
    rows, V = x.shape
    ld = ld or V
    wide = np.full((rows, ld), 1e30, np.float32)           # behind a row: never read as a value
    wide[:, :V] = x
    d = dict(x=DeviceArray.from_numpy(lib, wide), tok=DeviceArray.from_numpy(lib, np.asarray(tok, np.int32)))
    for k, n in (("lp", rows), ("rank", rows), ("ent", rows), ("top", rows * n_top), ("top_lp", rows * n_top)):
        d[k] = DeviceArray.from_numpy(lib, np.full(n + 4, -77, np.int32))
    need = lib.cgx_token_logprobs_ws(rows, V, n_top)
    ws = DeviceArray.from_numpy(lib, np.full(need + 64, 0xC3, np.uint8))
    p = lambda k: d[k].ptr if k in want else None          # noqa: E731
    rc = lib.cgx_token_logprobs_dev(d["x"].ptr, ld, rows, V, d["tok"].ptr if "lp" in want or "rank" in want else None,
                                    n_top, p("lp"), p("rank"), p("ent"), d["top"].ptr if n_top else None,
                                    d["top_lp"].ptr if n_top else None, ws.ptr, need)
    assert rc == 0, last_error(lib)
    assert lib.cgx_synchronize() == 0, last_error(lib)
    assert np.all(ws.numpy(np.uint8, (need + 64,))[need:] == 0xC3)
    out = {}
    for k, n, t, s in (("lp", rows, np.float32, (rows,)), ("rank", rows, np.int32, (rows,)),
                       ("ent", rows, np.float32, (rows,)), ("top", rows * n_top, np.int32, (rows, n_top)),
                       ("top_lp", rows * n_top, np.float32, (rows, n_top))):
        a = d[k].numpy(np.int32, (n + 4,))
        assert np.all(a[n:] == -77), k
        if k in ("lp", "rank", "ent") and k not in want:
            assert np.all(a == -77), k
        out[k] = a[:n].view(t).reshape(s)
    return out


def _reference(x, tok, n_top):
    rows, V = x.shape
    x = x.astype(np.float64)
    out = dict(lp=np.full(rows, -np.inf), rank=np.full(rows, V), ent=np.zeros(rows),
               top=np.full((rows, n_top), -1), top_lp=np.full((rows, n_top), -np.inf))
    for r in range(rows):
        v = x[r]
        bad = np.isnan(v).any() or np.isposinf(v).any() or np.isneginf(v).all()
        with np.errstate(invalid="ignore", divide="ignore"):
            m = v.max() if not bad else 0.0
            e = np.exp(v - m)
            z = e.sum()
            lp = v - m - np.log(z)
            if bad:
                lp = np.full(V, np.nan)
            t = e > 0
            out["ent"][r] = np.nan if bad else -np.sum(e[t] / z * lp[t])
        # NaN below everything, ties to the lowest index
        order = np.lexsort((np.arange(V), -np.where(np.isnan(v), -np.inf, v), np.isnan(v)))
        if 0 <= tok[r] < V:
            out["lp"][r] = lp[tok[r]]
            out["rank"][r] = int(np.argwhere(order == tok[r])[0, 0])
        n = min(n_top, V)
        out["top"][r, :n] = order[:n]
        out["top_lp"][r, :n] = lp[order[:n]]
    return out


def _close(a, e, tol):
    fin = np.isfinite(e)
    np.testing.assert_array_equal(a[~fin], e[~fin].astype(np.float32))
    assert np.all(np.abs(a[fin] - e[fin]) <= tol[fin]), float(np.max(np.abs(a[fin] - e[fin]) / tol[fin]))


def _check(got, exp):
    np.testing.assert_array_equal(got["rank"], exp["rank"])
    np.testing.assert_array_equal(got["top"], exp["top"])
    with np.errstate(invalid="ignore"):
        for k in ("lp", "top_lp"):
            _close(got[k], exp[k], 6e-6 + np.abs(exp[k]) * 2.0 ** -23)
        _close(got["ent"], exp["ent"], 6e-6 * (1 + np.abs(exp["ent"])))


@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 255, 257, 1000, 4095, 4096, 4097, 8191, 8193, 32000, 50257, 128256])
@pytest.mark.parametrize("rows,n_top", [(1, 0), (1, 5), (5, 20), (37, 32), (9, 1)])
def test_logprobs(gpu, V, rows, n_top):
    rng = np.random.default_rng(V + rows + n_top)
    if V > 30000 and rows > 9:
        rows = 9
    x = (rng.normal(size=(rows, V)) * rng.uniform(0.1, 4, (rows, 1))).astype(np.float32)
    tok = rng.integers(0, V, rows)
    tok[0] = int(x[0].argmax())
    _check(_run(gpu, x, tok, n_top, ld=V + 3), _reference(x, tok, n_top))


@pytest.mark.parametrize("V", [70, 5000, 40000])
def test_logprobs_of_ties_masks_and_bad_values(gpu, V):
    rng = np.random.default_rng(V)
    x = rng.normal(size=(14, V)).astype(np.float32)
    tok = rng.integers(0, V, 14)
    x[0] = 1.5                                             # all alike: the lowest indices, rank = index
    x[1] = np.round(x[1] * 2)                              # heavy ties
    x[2, rng.random(V) < 0.9] = -np.inf                    # masked tokens, the given one among them
    x[2, tok[2]] = -np.inf
    x[3] = -np.inf                                         # only one token left
    x[3, 17] = -3.0
    x[4] = -np.inf                                         # nothing left
    x[5, 9] = np.nan
    x[6, V - 1] = np.inf
    x[7] *= 1e-30
    x[8] = np.where(rng.random(V) < 0.5, 0.0, -0.0)        # equal values of both signs
    x[9, 3] = 90.0                                         # a row with one certain token
    x[10] = np.finfo(np.float32).min                       # the type's lowest value
    x[10, 20] = 0.0
    x[11] = np.nan
    tok[12], tok[13] = -1, V                               # no token of the vocabulary
    x[12] *= 30
    for n_top in (0, 7, 32):
        _check(_run(gpu, x, tok, n_top), _reference(x, tok, n_top))


def test_logprobs_outputs_may_be_left_out(gpu):
    rng = np.random.default_rng(3)
    x = rng.normal(size=(3, 9000)).astype(np.float32)
    tok = rng.integers(0, 9000, 3)
    full = _run(gpu, x, tok, 4)
    for want in (("lp",), ("rank",), ("ent",), ()):
        got = _run(gpu, x, tok, 4, want=want)
        for k in want + ("top", "top_lp"):
            np.testing.assert_array_equal(got[k], full[k])


def test_logprobs_agree_with_the_sampler_lists(gpu):
    """cgx_topk_lists_dev's order and probabilities (within its k): the same tokens, exp(logprob) renormalised."""
    rng = np.random.default_rng(5)
    rows, V, K = 4, 32000, 8
    x = rng.normal(size=(rows, V)).astype(np.float32) * 2
    got = _run(gpu, x, np.zeros(rows, int), K)
    dx = DeviceArray.from_numpy(gpu, x)
    li, lp = DeviceArray(gpu, rows * K * 4), DeviceArray(gpu, rows * K * 4)
    assert gpu.cgx_topk_lists_dev(dx.ptr, rows, V, K, 1.0, li.ptr, lp.ptr) == 0 and gpu.cgx_synchronize() == 0
    np.testing.assert_array_equal(got["top"], li.numpy(np.int32, (rows, K)))
    p = np.exp(got["top_lp"].astype(np.float64))
    np.testing.assert_allclose(p / p.sum(1, keepdims=True), lp.numpy(np.float32, (rows, K)), rtol=2e-5)
