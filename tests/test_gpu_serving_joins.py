"""GPU: rows of more pieces than a wave has lanes, which the joining launches
take in several rounds.

Tolerances: those of test_gpu_logprobs.py and test_gpu_paged.py.  They count the
32-bit roundings within a piece (8192 values, 384 keys over four waves), which
longer rows leave alone: log probabilities are joined in 64 bits, and the
attention's 100 pieces add 100 more terms to sums of at most 96 keys a wave."""
from __future__ import annotations

import numpy as np
import pytest

import paged_ref as R
import test_gpu_logprobs as logprobs

pytestmark = pytest.mark.gpu
TOL = 8e-6


@pytest.mark.parametrize("rows,V", [(7, 262144), (7, 262145), (7, 600000), (14, 600000)])
def test_logprobs_of_more_segments_than_lanes(gpu, rows, V):
    """Segments of 4096 values, 64, 65 and 147 of them, and 74 of 8192: ties, NaN and the largest values around the
    64th, where the second round begins with the list so far, and past the 127th."""
    rng = np.random.default_rng(V + rows)
    x = rng.normal(size=(rows, V)).astype(np.float32)
    tok = rng.integers(0, V, rows)
    edge = 63 * 4096
    x[1] = 1.5                                             # all alike: the lowest indices
    x[2, edge - 20:edge + 4096 + 20] = 7.0                 # equal values on both sides of the round's end
    tok[2] = edge + 4095
    x[3, [5, edge - 1, edge + 1, V - 1]] = np.nan
    x[3, edge - 40:edge - 20] = 6.0
    x[4] = -np.inf                                         # fewer numbers than alternatives, in the last segments
    x[4, [edge - 7, edge + 5, V - 9, V - 2]] = [1.0, 2.0, 3.0, 1.0]
    x[5, V - 50:] = np.arange(50) * 0.125 + 6              # the last segment has the whole list
    tok[5] = V - 1
    x[6] = np.float32(-np.inf)                             # nothing at all
    for n_top in (32, 5, 0):
        logprobs._check(logprobs._run(gpu, x, tok, n_top), logprobs._reference(x, tok, n_top))


def _same_key(b, to, of):
    """Key `to` of the first sequence becomes key `of`, its value stays."""
    P, at = b.P, lambda j: (0, int(b.table[0, j // b.P]))  # noqa: E731
    for a in (b.pool.k, b.pool.ks):
        a[at(to)][:, to % P] = a[at(of)][:, of % P]
    b.K[0][to] = b.K[0][of]


@pytest.mark.parametrize("H,Hk,D,gs", [(4, 1, 64, 64), (1, 1, 256, 256)])
def test_attention_of_more_pieces_than_lanes(gpu, H, Hk, D, gs):
    """104 pieces of one row's keys (64, the most, off the matrix cores), the largest score in an early piece, in a late
    one, and in both alike."""
    rng = np.random.default_rng(D)
    kv, early, late = 40001, 700, 39000
    b = R.Batch(gpu, rng, [kv], [4], 256, H, Hk, D, gs)
    _same_key(b, 39500, 900)
    K = b.K[0][:, 0].astype(np.float32)
    c = np.float32(16 / np.sqrt(D))                        # a score near 16, the others about 16 / sqrt(D) from 0
    b.q[0], b.q[1], b.q[2] = c * K[early], c * K[late], c * K[900]
    b.bind()
    need = gpu.cgx_attention_paged_ws(b.cache, b.step, H)
    assert need >= 64 * H * D * 4
    o, ls = b.attend(max_rows=4)
    O, L, A, F = b.reference()
    assert np.all(np.abs(o - O) <= TOL * A + F + 1e-37)
    assert np.all(np.abs(ls - L) <= TOL * (1 + np.abs(L)))
