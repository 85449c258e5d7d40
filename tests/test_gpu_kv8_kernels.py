"""Which kernel the 8-bit cache's attention runs, and that rotated queries keep what the header promises: 22 bits, but for the
tcgen05 kernel with head_dim 128 and round_q, which rounds them to fp16."""
import dataclasses

import numpy as np
import pytest
import torch

import kv8_plain as plain
from aihost_b200 import F16, F32, KV8_SPLIT_CACHE, KV8_TENSOR, ROPE_INTERLEAVED, ROPE_NEOX, ROPE_NONE
from aihost_b200.kv8 import Kv8Ops
from test_gpu_kv8 import ATTENDS, BOUNDS, DEV, World
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
@pytest.mark.parametrize("D, P, rounded", [(64, 16, False), (64, 16, True), (128, 64, False), (128, 64, True), (128, 16, False)])
def test_rotated_queries_keep_their_bits(ctx, D, P, rounded, cached, new, G, mode, max_kv):
    w = World(ctx, cached, new, Hq=2 * G, H=2, D=D, P=P, mode=mode, seed=61, theta=5e5, scale=1.5)
    w.spec = dataclasses.replace(w.spec, round_q=rounded)
    w.ops = Kv8Ops(ctx, w.spec)
    assert {_kernel(w, b) for b in BOUNDS} == _wanted(w)
    q = _q(w, lambda s: 0.5 + w.g.standard_normal(s))
    if _kernel(w, max_kv) == KV8_TENSOR and D == 128 and rounded:
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


@pytest.mark.parametrize("rounded", [False, True])
@pytest.mark.parametrize("what", ["cap", "bias", "documents", "chunks", "one row"])
@pytest.mark.parametrize("mode", [ROPE_INTERLEAVED, ROPE_NEOX])
def test_rotated_prompts_of_either_precision(ctx, mode, what, rounded):
    """head_dim 128, whose rings hold one tile of K and V or two: ranges longer than they hold, uneven ones, gaps between two
    query tiles' documents, and ranges cut into chunks."""
    cached, new = {"chunks": ([3300, 100], [90, 40]), "one row": ([700, 5], [1, 300])}.get(what, ([700, 0, 40], [300, 129, 17]))
    w = World(ctx, cached, new, Hq=8, H=1, D=128, P=32, mode=mode, cap=6.0 if what == "cap" else 0.0, seed=62)
    w.spec = dataclasses.replace(w.spec, round_q=rounded)
    w.ops = Kv8Ops(ctx, w.spec)
    first = slopes = None
    if what == "bias":
        slopes = [2.0 ** -(h + 1) for h in range(8)]
    if what == "documents":  # rows 0..15 of a sequence look back to its start, the later ones to their own neighbours
        first = [0 if i < 16 else max(0, int(p) - 20) for n, c in zip(new, cached) for i, p in enumerate(range(c, c + n))]
    most = 40000  # far enough for the tcgen05 kernel, in chunks
    assert _kernel(w, most) == KV8_TENSOR
    q, q64 = w.rows(w.Hq)
    out = w.attend(q.to(DEV), max_kv=most, first=first, slopes=slopes)
    again = w.attend(q.to(DEV), max_kv=most, first=first, slopes=slopes)
    torch.cuda.synchronize()
    ctx.sync_status()
    assert torch.equal(out, again)
    ref, weight, _ = plain.attend(q64, w.start, w.kv_len, w.table, w.P, w.k, w.v, w.ks, w.vs, w.scale, w.cap, w.theta, mode,
                                  first=first, slopes=None if slopes is None else np.float32(slopes))
    ds = (2.0 ** -11 if rounded else 2.0 ** -19) * _pair_size(w, q64)[..., None]
    tol = 2.0 ** -11 * np.abs(ref) + weight * (2.0 ** -11 + 2.0 ** -16 + 2 * ds) + 1e-7
    assert (np.abs(out.double().cpu().numpy() - ref) - tol).max() <= 0
