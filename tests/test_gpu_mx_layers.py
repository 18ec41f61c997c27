"""GPU: the transposed copy of a weight whose outputs are of very different sizes.  A chunk of 128 outputs has a layer for
each range of six powers of two that a block of 32 neighbours has values in, and none for the empty ranges between: what a
small row costs does not depend on how small it is.  Bounds of the gradients: those of test_gpu_mx.py."""
from __future__ import annotations

import numpy as np
import pytest

import mx_ref as R
from cogito_amd.capi import CGX_MX_FP32
from test_gpu_mx import Loss, Weight, _check, _rows, _up
from test_mx_api import Weight as Handle

pytestmark = pytest.mark.gpu


def _layers(c, b, V, K):
    """Layers of each chunk of 128 outputs, from codes [V][blocks][32] and bytes [V][blocks]."""
    held = (c.reshape(V, -1)[:, :K] & 7) != 0
    s = np.repeat(b, 32, 1)[:, :K].astype(int)
    out = []
    for n0 in range(0, V, 128):
        found = {0}
        for n in range(n0, min(n0 + 128, V), 32):
            h, e = held[n:min(n + 32, n0 + 128)], s[n:min(n + 32, n0 + 128)]
            fine = ~(e == 255).any(0)
            top = np.where(h, e, -1).max(0)
            at = (top - e) // 6
            found |= set(at[h & fine].tolist())
        out.append(len(found))
    return out


# rows of each chunk that are so many powers of two below the others, and the layers that makes (2, 5 and 13 beside 0 for the
# fourth, and 10 for 80 - 15 in the input that the small rows have to themselves)
@pytest.mark.parametrize("small,layers", [((), 1), ((60,), 2), ((100, 100), 2), ((15, 30, 80), 5), ((9, 10), 2)])
def test_layers_that_hold_nothing_are_left_out(gpu, small, layers):
    rng = np.random.default_rng(21)
    rows, K, V = 20, 70, 600
    # magnitudes between 0.25 and 0.5 of a row's power of two: each block's byte is the row's own
    w = rng.uniform(0.26, 0.49, (V, K)) * rng.choice([-1, 1], (V, K))
    for i, p in enumerate(small):
        w[5 + i::128] *= 2.0 ** -p
    # an input in which the small rows alone have values
    if small:
        alone = np.ones(V, bool)
        for i in range(len(small)):
            alone[5 + i::128] = False
        w[alone, 40] = 0
    c, b = R.quantise(w.astype(np.float32), 4)
    W = R.values(c, b, 4, K).T
    handle = Weight(gpu, R.pack(c, 4), b, K, V, grad=1)
    raw = Handle.from_address(handle.ptr)
    first = [raw.first[i] for i in range(raw.chunks128 + 1)]
    assert np.diff(first).tolist() == _layers(c, b, V, K) and raw.tchunks == first[-1]
    assert np.diff(first).tolist() == [layers] * 5
    h = _rows(rng, rows, K)
    t = rng.choice(np.concatenate([np.arange(5 + i, V, 128) for i in range(max(1, len(small)))]), rows).astype(np.int32)
    out = Loss(gpu, handle, h, t, CGX_MX_FP32, V).run()
    _check(out, h, W, t, CGX_MX_FP32)
    if small:
        assert np.all(out[2][:, 40] != 0)


def test_layers_over_the_whole_range(gpu):
    """Scales from 2 to 254 in 128 outputs: all 43 layers, 32 of them in one block.  The rows' logits stay small: hidden
    values are 0 in the inputs where the weight is large."""
    rows, K, V = 3, 64, 256
    c = np.full((V, 2, 32), 2, np.int64)                     # 1.0 over the block's scale
    b = np.full((V, 2), 127, np.uint8)
    n = np.arange(V)
    below = np.where(n // 32 % 2 == 0, n % 32, np.where(n % 32 > 0, n % 32 + 11, 0))
    b[:, 1] = 254 - 6 * below                                # layers 0 .. 31 and 0, 12 .. 42
    handle = Weight(gpu, R.pack(c, 4), b, K, V, grad=1)
    raw = Handle.from_address(handle.ptr)
    first = [raw.first[i] for i in range(raw.chunks128 + 1)]
    assert np.diff(first).tolist() == _layers(c, b, V, K) == [43, 43]
    h = np.zeros((rows, K), np.float32)
    h[:, 0] = [0.5, 0, -1]
    t = np.array([0, 100, 130], np.int32)
    loss, lse, dh = Loss(gpu, handle, h, t, CGX_MX_FP32, V).run()
    W = R.values(c, b, 4, K).T
    _check((loss, lse, dh), h, W, t, CGX_MX_FP32)


@pytest.mark.parametrize("K,V", [(40, 130), (300, 1000)])
def test_a_block_without_a_number_needs_no_layer(gpu, K, V):
    """A block with a byte of 255 reads as NaN whatever else it holds."""
    rng = np.random.default_rng(22)
    codes, b, _ = R.weight(rng, V, K)
    b = b.copy()
    b[40, 0], b[41, 0] = 255, 20                             # the second one far below its neighbours, in a block of NaN
    handle = Weight(gpu, codes, b, K, V, grad=1)
    raw = Handle.from_address(handle.ptr)
    c = R.unpack(codes, V, -(-K // 32), 4)
    assert np.diff([raw.first[i] for i in range(raw.chunks128 + 1)]).tolist() == _layers(c, b, V, K)
    assert raw.tchunks == raw.chunks128
