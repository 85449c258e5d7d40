"""The 4-bit cache's attention where its numbers leave the ordinary range. Bounds as in test_gpu_kv4.py, from the number formats;
results in fp32, so that nothing of an fp16 result's rounding hides what the weights lose."""
import dataclasses

import numpy as np
import pytest
import torch

import kv4_plain as plain4
import kv8_plain as plain
from aihost_b200 import F16, F32, KV8_TENSOR, ROPE_NEOX, ROPE_NONE
from aihost_b200.kv4 import Kv4Ops
from test_gpu_kv4 import World4
from test_gpu_kv8 import BOUNDS, DEV

pytestmark = pytest.mark.gpu


def _attend32(ctx, w, q, **kw):
    out = w.attend(q.to(DEV), ops=Kv4Ops(ctx, dataclasses.replace(w.spec, out_dtype=F32)), **kw).double().cpu().numpy()
    ctx.sync_status()
    return out


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("gap", [16, 20, 24, 30])
@pytest.mark.parametrize("D, P, new", [(64, 16, [64, 255]), (128, 128, [130, 255]), (128, 32, [1, 1])])
def test_small_weights_of_large_values(ctx, D, P, new, gap, biased, max_kv):
    """Rows 0 and 140 take nearly all the weight and hold next to nothing; the others have 2^-gap of it, and all of the result: their
    weights keep fp16's bits, whichever row has the largest score."""
    w = World4(ctx, [300, 30], new, Hq=4, H=2, D=D, P=P, scale=1.0 / D, seed=gap)
    q = torch.from_numpy(w.g.uniform(0.5, 1.5, (w.T, w.Hq, D))).half()  # with K alike in all elements: score = its value, about
    shape = w.ks.shape[:-1]
    low = -gap * np.log(2) - w.g.uniform(0, 0.5, shape)
    w.ks = np.stack([low, np.full(shape, 2.0 ** -10)], -1).astype(np.float16)
    step = 512.0 * 2.0 ** -w.g.integers(0, 5, shape)
    w.vs = np.stack([-7.5 * step, step], -1).astype(np.float16)
    for b, length in enumerate(w.kv_len):
        for t in (0, 140):
            if t < length:
                at = w.table[b][t // P], slice(None), t % P
                w.ks[at] = np.float16([0.0, 2.0 ** -10])
                w.vs[at] = np.float16([0.0, 2.0 ** -24])
    slopes = [2.0 ** -(12 + h) for h in range(w.Hq)] if biased else None
    got = _attend32(ctx, w, q, slopes=slopes, max_kv=max_kv)
    ref, off, most, size = w.reference(q.double().numpy(), slopes=slopes)
    tol = off * 2.0 ** -11 + most * (2.0 ** -16 + 2.0 ** -18 * size[..., None])
    assert (np.abs(got - ref) <= tol).all(), (np.abs(got - ref) / tol).max()
    if max(new) > 16 and max_kv:
        assert w.ops.plan(len(new), w.T, max(new), max_kv)[1] == KV8_TENSOR


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("D, P", [(64, 16), (128, 64)])
def test_steps_of_either_sign(ctx, D, P, io, max_kv):
    """An append makes none below zero, but a code stands for low + step * c whatever the step's sign."""
    w = World4(ctx, [150, 9], [30, 70], Hq=4, H=2, D=D, P=P, io=io, seed=19)
    for r in (w.ks, w.vs):
        r[..., 1] *= w.g.choice(np.float16([-1, 1]), r.shape[:-1])
    w.check(ctx, max_kv=max_kv)
    w.check(ctx, max_kv=max_kv, slopes=[2.0 ** -(h + 1) for h in range(4)])


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("D, P", [(64, 16), (128, 128)])
def test_infinite_ranges_of_keys(ctx, D, P, io, max_kv):
    """Values without bound times a q of both signs are no number: such a row of K makes one of the rows that see it, and does
    nothing to those that do not."""
    w = World4(ctx, [100, 33], [1, 40], P=P, D=D, io=io, mode=ROPE_NONE, seed=4)
    first = [64] + [48 if p >= 48 else 0 for p in w.pos[1:]]
    q, _ = w.rows(w.Hq)
    hit = torch.tensor([b == 1 and p < 48 for b, p in zip(np.repeat([0, 1], w.new), w.pos)])
    keep = w.ks.copy()
    for col, bad in ((0, np.inf), (0, -np.inf), (1, np.inf), (1, -np.inf)):
        w.ks = keep.copy()
        w.ks[w.table[1][0], :, 3, col] = bad  # row 3 of sequence 1: seen by its first document's rows only
        w.k[w.table[1][0], :, 3] |= 0x11      # no code 0, whose value would be low alone
        out = w.attend(q.to(DEV), first=first, max_kv=max_kv).cpu()
        ctx.sync_status()
        assert torch.isnan(out[hit]).all() and torch.isfinite(out[~hit]).all()


def test_append_of_values_beyond_fp16(ctx):
    """A finite row whose low and step are fp16 numbers is stored, however large its values: to the bit, in fp32 within half a step of
    them, its own rounding and those of low and step; read as fp16 what passes its range is infinite."""
    w = World4(ctx, [0], [40], Hq=2, H=2, D=64, io=F32, seed=8)
    top = np.float32([65520.0, 1e5, 6e5, 9e5, 1e6, 1e30])
    k, v = (torch.from_numpy(w.g.uniform(0, 1, (w.T, 2, 64)).astype(np.float32)) for _ in range(2))
    k *= torch.from_numpy(np.resize(top, w.T))[:, None, None]
    k[..., 0], k[..., 1] = 0.0, torch.from_numpy(np.resize(top, w.T))[:, None]
    pools = w.pools()
    w.ops.append(k.to(DEV), v.to(DEV), w.dev(w.slots), None, *pools)
    codes, low, step = plain4.quantise(k.numpy())
    at = w.slots // w.P, slice(None), w.slots % w.P
    assert np.array_equal(pools[2].cpu().numpy()[at], np.stack([low, step], -1), equal_nan=True)
    assert np.array_equal(pools[0].cpu().numpy()[at], plain4.pack(codes))
    slots = w.dev(w.slots)
    got32, got16 = (w.ops.read(pools[0], pools[2], slots, t).double().cpu().numpy() for t in (torch.float32, torch.float16))
    ctx.sync_status()
    fine = np.resize(top <= 9e5, w.T)  # 1e6 / 15 passes fp16's range
    x = k.double().numpy()
    assert np.isnan(got32[~fine]).all() and np.isnan(got16[~fine]).all()
    # half a step; codes stop at 15, and the step was rounded: 15 * 2^-11 of it
    assert (np.abs(got32 - x)[fine] <= step.astype(float)[fine][..., None] * (0.5 + 15 * 2.0 ** -11 + 2.0 ** -16)).all()
    assert np.array_equal(np.isinf(got16[fine]), np.abs(got32[fine]) >= 65520.0)


@pytest.mark.parametrize("D, Hq, cached, new", [(128, 4, [30000, 17000], [1, 1]), (64, 4, [30000], [1]), (128, 16, [20000], [2]), (64, 16, [9000], [9])])
def test_fp32_results_over_long_caches(ctx, D, Hq, cached, new):
    """Thousands of rows of codes whose mean is 7.5: the error, in root mean square, does not grow with them. Of the result: weights
    2^-22 from ex2 and their pairs, scores of about 1 in eight products 2^-22, a step's sums in eight more 2^-22, a warp's
    2^8 additions to O 2^-24 * 2^4 at random, 2^-20 at most together."""
    w = World4(ctx, cached, new, Hq=Hq, H=4, D=D, P=128, io=F32, seed=D)
    q, q64 = w.rows(w.Hq)
    got = w.attend(q.to(DEV)).double().cpu().numpy()
    ctx.sync_status()
    ref = w.reference(q64)[0]
    assert np.sqrt(((got - ref) ** 2).mean()) <= 2.0 ** -20 * np.sqrt((ref ** 2).mean())


@pytest.mark.parametrize("D, mode", [(64, ROPE_NONE), (128, ROPE_NEOX)])
def test_prompts_over_long_caches(ctx, D, mode):
    """Blocks that walk 250 tiles of codes 6 to 9, whose mean is 7.5. The error, in root mean square, is that of rounding the result and the weights to
    fp16, each 2^-11 / sqrt(3) * sqrt(0.541) = 0.425 * 2^-11 (of a number anywhere in its binade), 0.60 * 2^-11 together."""
    new, cached, G, P = 2048, 30000, 4, 128
    w = World4(ctx, [cached], [new], Hq=8 * G, H=8, D=D, P=P, mode=mode, seed=D)
    w.v = (w.v & 0x33) + 0x66
    w.vs[..., 0] = -7.5 * w.vs[..., 1].astype(np.float32)
    q, q64 = w.rows(w.Hq)
    got = w.attend(q.to(DEV)).double().cpu()
    ctx.sync_status()
    assert w.ops.plan(1, new, new, cached + new)[1] == KV8_TENSOR
    pages, rows = w.table[0][:-(-(cached + new) // P)], np.arange(0, new, 37)
    turned = plain.rotate(q64[rows], cached + rows, w.theta, mode)
    err = size = 0.0
    for h, g in ((0, 1), (5, 22)):
        k, v = (torch.from_numpy(plain4.values(p[pages, h], r[pages, h], np.float64).reshape(-1, D)[:cached + new]) for p, r in ((w.k, w.ks), (w.v, w.vs)))
        x = torch.from_numpy(turned[:, g]) @ k.T * w.scale
        x = x.masked_fill(torch.arange(cached + new)[None] > torch.from_numpy(cached + rows)[:, None], -torch.inf).softmax(-1) @ v
        err, size = err + ((got[rows, g] - x) ** 2).sum().item(), size + (x ** 2).sum().item()
    assert np.sqrt(err / size) <= 0.65 * 2.0 ** -11
