"""Which kernel the 8-bit cache's attention runs, and that rotated queries keep what the header says of it: 22 bits, but for the
tcgen05 kernel with head_dim 128, which rounds them to fp16."""
import numpy as np
import pytest

import kv8_plain as plain
from aihost_b200 import F16, F32, KV8_SPLIT_CACHE, KV8_TENSOR, ROPE_INTERLEAVED, ROPE_NEOX, ROPE_NONE
from test_gpu_kv8 import ATTENDS, BOUNDS, World
from test_gpu_kv8_range import _check, _q

pytestmark = pytest.mark.gpu


def _kernel(w, max_kv):
    return w.ops.plan(len(w.new), w.T, max(w.new), max_kv or int(w.kv_len.max()))[1]


def _wanted(w):
    """Between them the bounds run both kernels where both can: fp16 tensors, and more query rows a sequence than the
    split-cache kernel's tile has."""
    both = w.io == F16 and max(w.new) * (w.Hq // w.H) > 16
    return {KV8_SPLIT_CACHE, KV8_TENSOR} if both else {KV8_SPLIT_CACHE}


def _pair_size(w, q):
    """Per row and head: the largest, over a visible row, of scale * sum |k| (|x| + |y|), (x, y) the pair that an element is
    turned from. The rotation's fp32 sines, cosines and products are off by 2^-22 of that, the sums by 2^-19 of
    less."""
    a = np.abs(q)
    if w.mode == ROPE_INTERLEAVED:
        pair = np.repeat(a[..., 0::2] + a[..., 1::2], 2, axis=-1)
    else:
        half = a[..., :w.D // 2] + a[..., w.D // 2:]
        pair = np.concatenate([half, half], axis=-1)
    out, G = np.zeros(q.shape[:2]), w.Hq // w.H
    for b in range(len(w.new)):
        t0, t1, L = int(w.start[b]), int(w.start[b + 1]), int(w.kv_len[b])
        pages = w.table[b][:-(-L // w.P)]
        for h in range(w.H):
            k = (np.abs(w.k[pages, h].astype(float)) * w.ks[pages, h, None, None]).reshape(-1, w.D)[:L]
            for i, t in enumerate(range(t0, t1)):
                seen = k[:L - (t1 - t0) + i + 1]
                for g in range(h * G, h * G + G):
                    out[t, g] = w.scale * (seen @ pair[t, g]).max()
    return out


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("mode", [ROPE_INTERLEAVED, ROPE_NEOX])
@pytest.mark.parametrize("cached, new, G", [([300, 1029], [1, 1], 4), ([333], [1], 16), ([300, 77], [3, 2], 4),
                                            ([90, 0, 17], [60, 130, 1], 4), ([1500], [40], 7)])
@pytest.mark.parametrize("D, P", [(64, 16), (128, 64)])
def test_rotated_queries_keep_their_bits(ctx, D, P, cached, new, G, mode, max_kv):
    w = World(ctx, cached, new, Hq=2 * G, H=2, D=D, P=P, mode=mode, seed=61, theta=5e5, scale=1.5)
    kernel = _kernel(w, max_kv)
    assert {_kernel(w, b) for b in BOUNDS} == _wanted(w)
    q = _q(w, lambda s: 0.5 + w.g.standard_normal(s))
    if kernel == KV8_TENSOR and D == 128:
        _check(ctx, w, q, out_dtype=F32, max_kv=max_kv, ds=2.0 ** -11)
        return
    size = _pair_size(w, q)
    _, ref = _check(ctx, w, q, out_dtype=F32, max_kv=max_kv, size=size)
    # a rotated q that had lost the lower half of its pairs would not have passed
    turned = np.concatenate([plain.rotate(q[t0:t1], np.arange(L - (t1 - t0), L), w.theta, mode)
                             for t0, t1, L in zip(w.start, w.start[1:], w.kv_len)])
    lost, weight, _ = plain.attend(turned.astype(np.float16).astype(float), w.start, w.kv_len, w.table, P, w.k, w.v, w.ks,
                                   w.vs, w.scale, mode=ROPE_NONE)
    tol = weight * (2.0 ** -11 + 2.0 ** -16 + 2.0 ** -18 * size[..., None]) + 1e-7
    assert (np.abs(lost - ref) > tol).any()


@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("case", list(ATTENDS))
def test_the_bounds_choose_the_kernel(ctx, case, io):
    """What the two bounds of the attention tests are for."""
    w = World(ctx, io=io, **ATTENDS[case])
    assert {_kernel(w, b) for b in BOUNDS} == _wanted(w)
