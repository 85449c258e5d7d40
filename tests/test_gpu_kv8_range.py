"""The 8-bit cache's attention where its numbers leave the ordinary range: K with one large channel, q and V far from 1, V
scales far apart, caps far above the scores, scores far below zero, the loosest bounds. Bounds as in test_gpu_kv8.py, from the
number formats; every comparison is against the 64-bit form."""
import dataclasses

import numpy as np
import pytest
import torch

import kv8_plain as plain
from aihost_b200 import F16, F32, ROPE_INTERLEAVED, ROPE_NEOX, ROPE_NONE
from aihost_b200.kv8 import Kv8Ops
from test_gpu_kv8 import BOUNDS, DEV, World, _dt

pytestmark = pytest.mark.gpu


def _check(ctx, w, q, out_dtype=None, ds=2.0 ** -19, first=None, max_kv=None, tiny=1e-7, size=None):
    """Attention of q (float64, exact in the io type) on the GPU against the plain form. A score's error is `ds` of
    sum |q k| (or of `size`); weights rounded to fp16 are off by 2^-11, pairs of fp16 by 2^-18; an fp16 result by 2^-11 of itself."""
    ops = w.ops
    if out_dtype is not None:
        ops = Kv8Ops(ctx, dataclasses.replace(w.spec, out_dtype=out_dtype))
    qd = torch.from_numpy(q).to(_dt(w.io))
    assert torch.equal(qd.double(), torch.from_numpy(q))
    got = w.attend(qd.to(DEV), first=first, max_kv=max_kv, ops=ops)
    torch.cuda.synchronize()
    ctx.sync_status()
    ref, weight, own = plain.attend(q, w.start, w.kv_len, w.table, w.P, w.k, w.v, w.ks, w.vs, w.scale, w.cap, w.theta, w.mode,
                                    first=first)
    size = own if size is None else size
    tol = weight * ((2.0 ** -11 + 2.0 ** -16 if w.io == F16 else 2.0 ** -18) + 2 * ds * size[..., None]) + tiny
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -11 * np.abs(ref)
    got = got.double().cpu().numpy()
    over = np.abs(got - ref) - tol
    assert np.isfinite(got).all() and over.max() <= 0, (over.max(), np.unravel_index(over.argmax(), over.shape))
    return got, ref


def _q(w, draw):
    """Query rows from draw(shape), rounded to the io type, as float64."""
    return torch.from_numpy(np.ascontiguousarray(draw((w.T, w.Hq, w.D)))).to(_dt(w.io)).double().numpy()


STEPS = {"decode": dict(cached=[300, 1029], new=[1, 1], P=64), "few": dict(cached=[300, 77], new=[3, 2], P=32),
         "prompt": dict(cached=[90, 0], new=[60, 130], P=32)}


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("mode", [ROPE_NONE, ROPE_INTERLEAVED])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("step", list(STEPS))
def test_keys_with_one_large_channel(ctx, step, D, mode, io, max_kv):
    """One channel takes all of a page's int8 range and the others hold -1, 0 and 1; q is near 1 (all of one sign) and 0 in that
    channel: what a conversion with an offset would have to cancel is a thousand times the score."""
    w = World(ctx, D=D, io=io, mode=mode, seed=41, **STEPS[step])
    w.k = w.g.integers(-1, 2, w.k.shape).astype(np.int8)
    w.k[..., 0] = 127
    w.k[..., 1] = 127
    w.ks = w.g.uniform(2.5, 3.5, w.ks.shape).astype(np.float32) * np.float32(np.sqrt(128 / D))
    q = _q(w, lambda s: 1 + 0.3 * w.g.standard_normal(s))
    q[..., :2] = 0  # the first pair of the rotation
    _check(ctx, w, q, ds=2.0 ** -11 if io == F16 and mode != ROPE_NONE else 2.0 ** -19, max_kv=max_kv)


@pytest.mark.parametrize("mode", [ROPE_NONE, ROPE_INTERLEAVED, ROPE_NEOX])
@pytest.mark.parametrize("std", [3e-33, 1e-20, 1e-6, 1e-3, 1e4, 1e6, 1e30])
@pytest.mark.parametrize("step", list(STEPS))
def test_fp32_queries_of_any_size(ctx, step, std, mode):
    """fp32 q enters as a pair of fp16 with 22 bits whatever its size."""
    w = World(ctx, io=F32, mode=mode, scale=float(np.float32(0.1 / std)), seed=42, Hq=8, H=2, **STEPS[step])
    w.scale = float(np.float32(0.1 / std))
    rows = np.exp(w.g.uniform(-1, 1, (w.T, w.Hq, 1)))  # rows of unequal size
    _check(ctx, w, _q(w, lambda s: std * rows * w.g.standard_normal(s)), tiny=1e-9)


@pytest.mark.parametrize("step", list(STEPS))
def test_fp32_rows_of_zeros_and_of_unequal_elements(ctx, step):
    w = World(ctx, io=F32, seed=43, scale=1e-4, **STEPS[step])
    q = _q(w, lambda s: w.g.standard_normal(s) * np.exp(w.g.uniform(np.log(1e-3), np.log(1e6), s)))
    q[0] = 0
    got, ref = _check(ctx, w, q, tiny=1e-9)
    assert np.abs(ref[0]).max() > 0


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("mode", [ROPE_INTERLEAVED, ROPE_NEOX])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("step", list(STEPS))
def test_fp16_queries_whose_rotation_passes_the_range_of_fp16(ctx, step, D, mode, max_kv):
    """Elements up to 65504 turn into ones up to 92 K, which are no fp16."""
    w = World(ctx, D=D, mode=mode, scale=2e-6, seed=44, **STEPS[step])
    q = _q(w, lambda s: np.where(w.g.random(s) < 0.5, 1, -1) * w.g.uniform(50000, 65504, s))
    _check(ctx, w, q, ds=2.0 ** -11, max_kv=max_kv)


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("top", [1e-33, 3e-36, 2e-37])
@pytest.mark.parametrize("step", list(STEPS))
def test_tiny_values(ctx, step, top, io, max_kv):
    """V scales down to the least normal fp32 numbers: results of that size, not NaN."""
    w = World(ctx, D=128, io=io, seed=45, **STEPS[step])
    w.vs = w.g.uniform(top / 10, top, w.vs.shape).astype(np.float32)
    # below the least normal number, 1.2e-38, a result may be flushed
    got, ref = _check(ctx, w, _q(w, w.g.standard_normal), out_dtype=F32, max_kv=max_kv, tiny=1.2e-38)
    assert np.abs(ref).max() > 2 * top


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("io, low, high", [(F16, 1e-3, 500.0), (F16, 1e-9, 1e3), (F32, 1e-3, 500.0), (F32, 1e-9, 1e9)])
@pytest.mark.parametrize("D, P", [(64, 16), (128, 32)])
@pytest.mark.parametrize("cached", [[256, 0], [250, 2]])  # the second: edges inside tiles of 4 tokens too
def test_documents_whose_values_differ_in_size(ctx, cached, D, P, io, low, high, max_kv):
    """Rows of one document see nothing of another's values, nor of their size."""
    w = World(ctx, cached, [150, 200], D=D, P=P, io=io, seed=46)
    # at page edges: every page in one document
    edges = {0: [0, 64, 288, 320, cached[0] + 150], 1: [0, 96, 128, cached[1] + 200]}
    first = np.zeros(w.T, int)
    for b, e in edges.items():
        for i, (lo, hi) in enumerate(zip(e, e[1:])):
            w.vs[w.table[b][lo // P:-(-hi // P)]] *= (high if i % 2 else low) / 0.01
        for t in range(w.start[b], w.start[b + 1]):
            first[t] = max(x for x in e if x <= w.pos[t])
    _check(ctx, w, _q(w, w.g.standard_normal), out_dtype=F32, first=first.tolist(), max_kv=max_kv, tiny=1e-30)


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("step", list(STEPS))
def test_values_far_apart_in_sight_of_each_other(ctx, step, io, max_kv):
    """A few pages with values a million times the others', whose keys lie so far off that they add nothing."""
    w = World(ctx, D=128, io=io, seed=47, **STEPS[step])
    w.vs *= np.float32(1e-2)
    q = _q(w, lambda s: 0.5 + 0.1 * w.g.standard_normal(s))
    for b in range(len(w.new)):
        page = w.table[b][0]
        w.k[page] = -100  # scores about -100 * 0.1 * 0.5 * 128 / sqrt(128)
        w.ks[page] = 0.1
        w.vs[page] = 1e3
    _check(ctx, w, q, out_dtype=F32, max_kv=max_kv, tiny=1e-12)


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("cap", [1e3, 1e5])
@pytest.mark.parametrize("step", list(STEPS))
def test_caps_far_above_the_scores(ctx, step, cap, io, max_kv):
    """A capped score is as exact as an uncapped one: its error goes by the score, not by the cap."""
    w = World(ctx, D=128, io=io, cap=cap, seed=48, **STEPS[step])
    _check(ctx, w, _q(w, w.g.standard_normal), max_kv=max_kv)


@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("step", list(STEPS))
def test_scores_near_and_far_from_a_large_cap(ctx, step, io):
    """The same where single keys lie beyond the cap, so that no step of the cache is all small."""
    w = World(ctx, D=128, io=io, cap=1000.0, seed=49, **STEPS[step])
    q = _q(w, lambda s: np.abs(w.g.standard_normal(s)) + 0.5)
    w.k[:, :, ::8] = -127
    w.ks[:] = 0.02
    w.ks[::3] = 1.5  # -127 * 1.5 * 1.3 * 128 / sqrt(128): beyond the cap
    for b in range(len(w.new)):
        w.ks[w.table[b][0]] = 0.02
    w.k[:, :, ::8] = -127
    _check(ctx, w, q, ds=2.0 ** -18)


@pytest.mark.parametrize("step", list(STEPS))
def test_scores_below_every_sentinel(ctx, step):
    """All scores of a row at -1e31 and below: the largest still takes the row."""
    w = World(ctx, D=64, io=F32, scale=1e12, seed=50, **STEPS[step])
    q = _q(w, lambda s: np.full(s, 1e17))
    w.k[:] = w.g.integers(-120, -100, w.k.shape)
    w.ks[:] = 1.0
    best = [int(w.table[b][0]) for b in range(len(w.new))]
    for page in best:
        w.k[page, :, 0] = -10
    got, ref = _check(ctx, w, q, ds=0.0, tiny=1e-9)
    assert np.abs(ref).max() > 0.1


@pytest.mark.parametrize("max_kv", [2 ** 31 - 1, 2 ** 31 - 200, 2 ** 30])
@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("step", list(STEPS))
def test_the_loosest_bound(ctx, step, io, max_kv):
    """max_kv is any bound, up to the largest int32."""
    w = World(ctx, D=64, io=io, seed=51, **STEPS[step])
    _check(ctx, w, _q(w, w.g.standard_normal), max_kv=max_kv)


@pytest.mark.parametrize("cap", [0.0, 300.0])
@pytest.mark.parametrize("D", [64, 128])
def test_keys_on_either_side_of_the_rule_for_small_pages(ctx, D, cap):
    """Page scales spread over four powers of ten, in rounds of 32 blocks of rows: some pages' keys are converted one way, some
    the other, and a round of large ones follows a round of small ones."""
    w = World(ctx, D=D, P=16, Hq=4, H=2, cap=cap, seed=52, cached=[2500, 700], new=[1, 1])
    w.k = w.g.integers(-1, 2, w.k.shape).astype(np.int8)
    w.ks = np.exp(w.g.uniform(np.log(3e-4), np.log(3), w.ks.shape)).astype(np.float32)
    for b, n in enumerate(w.kv_len):
        order = np.argsort(w.ks[w.table[b][:-(-int(n) // 16)], 0])
        w.ks[w.table[b][:len(order)]] = w.ks[w.table[b][order]]  # small ones first
    _check(ctx, w, _q(w, lambda s: 1 + 0.3 * w.g.standard_normal(s)))


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("cap", [3.4e38, 1e36, 1e29, 1e-29, 1e-36, 1e-42])
@pytest.mark.parametrize("step", list(STEPS))
def test_caps_of_any_size(ctx, step, cap, io, max_kv):
    """The largest caps leave the scores as they are, the smallest make every visible row count alike."""
    w = World(ctx, D=64, io=io, cap=cap, seed=53, **STEPS[step])
    _check(ctx, w, _q(w, w.g.standard_normal), max_kv=max_kv)
