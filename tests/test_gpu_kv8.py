"""The 8-bit paged cache on the GPU against plain 64-bit forms (tests/kv8_plain.py).

Bounds, from the number formats:
  append     a stored value is the nearest integer to its target (within 1e-3 of the tie, for the fp32 arithmetic and
             the rotation's fp32 sine and cosine), its page's scale within 2^-20
  attention  fp16: the output's rounding 2^-11 |o|; P's rounding 2^-11 of sum p|v|; the score's error ds shifts p by up to
             2 ds, ds = 2^-11 of sum |q k| where a rotated q is rounded to fp16, else 2^-19 of it (fp32 sums, ex2)
             fp32: pairs of fp16 hold 22 bits; ex2.approx and fp32 sums 2^-18 of sum p|v| and 2^-19 of sum |q k|
"""
import dataclasses

import numpy as np
import pytest
import torch

import aihost_b200 as A
import kv8_plain as plain
from aihost_b200 import F16, F32, ROPE_INTERLEAVED, ROPE_NEOX, ROPE_NONE, AttnError
from aihost_b200.kv8 import Kv8Cache, Kv8Ops, Kv8Spec

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
I32 = torch.int32


def _dt(code):
    return torch.float16 if code == F16 else torch.float32


class World:
    """A pool with scattered pages, filled with int8 noise, and a step of new rows on top."""

    def __init__(self, ctx, cached, new, Hq=8, H=2, D=64, P=16, io=F16, mode=ROPE_NONE, cap=0.0, scale=0.0, seed=0, spare=3,
                 theta=10000.0):
        self.g = np.random.default_rng(seed)
        self.cached, self.new, self.P, self.D, self.H, self.Hq, self.io = cached, new, P, D, H, Hq, io
        self.mode, self.theta, self.cap = mode, theta, cap
        after = [-(-(c + n) // P) for c, n in zip(cached, new)]
        self.n_pages, self.max_pages = sum(after) + spare, max(after) + 1
        order = self.g.permutation(self.n_pages)
        self.table, at = np.full((len(cached), self.max_pages), -1), 0
        for b, n in enumerate(after):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.spec = Kv8Spec(Hq, H, D, P, self.n_pages, self.max_pages, io, io, scale, cap, theta, mode)
        self.scale = scale or float(np.float32(1) / np.sqrt(np.float32(D)))
        self.ops = Kv8Ops(ctx, self.spec)
        shape = (self.n_pages, H, P, D)
        self.k, self.v = (self.g.integers(-127, 128, shape).astype(np.int8) for _ in range(2))
        self.ks, self.vs = (self.g.uniform(0.002, 0.03, shape[:2]).astype(np.float32) for _ in range(2))
        self.start = np.concatenate([[0], np.cumsum(new)]).astype(np.int64)
        self.kv_len = np.array(cached) + np.array(new)
        self.pos = np.concatenate([np.arange(c, c + n) for c, n in zip(cached, new)] + [np.zeros(0, int)]).astype(np.int64)
        seq = np.repeat(np.arange(len(new)), new)
        self.slots = self.table[seq, self.pos // P] * P + self.pos % P
        self.T = int(self.start[-1])

    def rows(self, heads, std=1.0):
        x = torch.from_numpy(self.g.normal(0, std, (self.T, heads, self.D))).to(_dt(self.io))
        return x, x.double().numpy()

    def dev(self, x, dt=None):
        t = torch.from_numpy(np.ascontiguousarray(x))
        return t.to(dt or t.dtype).to(DEV)

    def attend(self, q, max_new=None, max_kv=None, prefix=None, first=None, slopes=None, ops=None):
        return (ops or self.ops).attend(
            q, self.dev(self.start, I32), self.dev(self.kv_len, I32), self.dev(self.table, I32), self.dev(self.k), self.dev(self.v),
            self.dev(self.ks), self.dev(self.vs), max_new or max(self.new), max_kv or int(self.kv_len.max()),
            prefix_len=None if prefix is None else self.dev(np.array(prefix), I32),
            row_first=None if first is None else self.dev(np.array(first), I32),
            alibi_slopes=None if slopes is None else self.dev(np.array(slopes), torch.float32))

    def check(self, ctx, std=1.0, prefix=None, first=None, slopes=None, **kw):
        q, q64 = self.rows(self.Hq, std)
        out = self.attend(q.to(DEV), prefix=prefix, first=first, slopes=slopes, **kw)
        torch.cuda.synchronize()
        ctx.sync_status()
        ref, weight, size = plain.attend(q64, self.start, self.kv_len, self.table, self.P, self.k, self.v, self.ks, self.vs,
                                         self.scale, self.cap, self.theta, self.mode, prefix, first,
                                         None if slopes is None else np.float32(slopes))
        got = out.double().cpu().numpy()
        assert got.shape == ref.shape
        rounded_q = self.io == F16 and self.mode != ROPE_NONE
        ds = size[..., None] * (2.0 ** -11 if rounded_q else 2.0 ** -19)
        if self.io == F16:
            tol = 2.0 ** -11 * np.abs(ref) + weight * (2.0 ** -11 + 2.0 ** -16 + 2 * ds) + 1e-7
        else:
            tol = weight * (2.0 ** -18 + 2 * ds) + 1e-9
        over = np.abs(got - ref) - tol
        assert np.isfinite(got).all() and over.max() <= 0, (over.max(), np.unravel_index(over.argmax(), over.shape))
        return got


# ------------------------------------------------------------------------------------------------ page maps

def _map(ctx, P, n_pages, max_pages, max_tokens, cached, new, seed=0, in_place=False, free=None):
    g = np.random.default_rng(seed)
    order = g.permutation(n_pages)
    table, at = np.full((len(cached), max_pages), -1), 0
    for b, c in enumerate(cached):
        n = -(-c // P)
        table[b, :n] = order[at:at + n]
        at += n
    stack = np.concatenate([order[at:], order[:at]])
    count = n_pages - at if free is None else free
    want = plain.page_map(P, n_pages, max_pages, max_tokens, cached, new, stack.tolist(), count, table.tolist())
    ops = Kv8Ops(ctx, Kv8Spec(8, 2, 64, P, n_pages, max_pages))
    t = lambda x: torch.tensor(x, dtype=I32, device=DEV)  # noqa: E731
    d_table, d_len, d_free = t(table), t(cached), t([count])
    into = None
    if in_place:
        from aihost_b200.kv8 import StepMap

        into = StepMap(d_len, t([7] * (len(cached) + 1)), torch.full((max_tokens,), 7, dtype=torch.int64, device=DEV),
                       t([7] * max_tokens), d_free)
    m = ops.map_pages(d_len, t(new), t(stack), d_free, d_table, max_tokens, into=into)
    torch.cuda.synchronize()
    got = (d_table.tolist(), m.kv_len.tolist(), m.row_start.tolist(), m.slots.tolist(), m.positions.tolist(),
           m.free_count.item())
    assert got == want[:6]
    return want[6]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("P, batch, hi, new_hi, spare", [
    (16, 1, 0, 1, 0), (16, 1, 15, 40, 3), (32, 7, 100, 3, 1), (64, 64, 8000, 1, 0), (128, 300, 900, 9, 100),
    (16, 2000, 50, 60, 5000), (64, 8192, 20, 2, 0)])
def test_page_map_matches_plain(ctx, P, batch, hi, new_hi, spare, in_place):
    g = np.random.default_rng(batch + P)
    cached, new = g.integers(0, hi + 1, batch).tolist(), g.integers(0, new_hi + 1, batch).tolist()
    if new_hi == 1:
        new = [1] * batch
    n_pages = sum(-(-(c + n) // P) for c, n in zip(cached, new)) + 2
    max_pages = -(-(hi + new_hi) // P) + 1
    assert not _map(ctx, P, n_pages, max_pages, sum(new) + spare, cached, new, in_place=in_place)
    ctx.sync_status()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kw, status", [
    (dict(cached=[15, 16], new=[2, 1], free=1), A.ENOMEM),
    (dict(cached=[15, 16], new=[2, -1]), A.EINVAL),
    (dict(cached=[15, 16], new=[2, 20]), A.EINVAL),            # more tokens than max_tokens
    (dict(cached=[15, 16], new=[2, 2 ** 31 - 17]), A.EINVAL),  # a sum past 2^31
    (dict(cached=[63, 16], new=[2, 1]), A.EINVAL),             # beyond max_pages
    (dict(cached=[15, 16], new=[2, 1], free=999), A.EINVAL),
    (dict(cached=[15] * 3000, new=[2] * 3000, max_tokens=6000, free=2999), A.ENOMEM),
])
def test_page_map_refuses_a_step_whole(ctx, kw, status, in_place):
    kw = dict(kw)
    cached, new = kw.pop("cached"), kw.pop("new")
    assert _map(ctx, 16, 40 + len(cached) * 2, 4, kw.pop("max_tokens", 10), cached, new, in_place=in_place, **kw)
    with pytest.raises(AttnError) as e:
        ctx.sync_status()
    assert e.value.status == status
    ctx.sync_status()  # read and cleared


def test_pages_go_round(ctx):
    """Steps and releases against the plain map: no page in two hands, none lost, reused pages begun anew."""
    P, batch, n_pages, max_pages = 16, 9, 40, 12
    g = np.random.default_rng(3)
    cache = Kv8Cache(ctx, Kv8Spec(4, 2, 64, P, n_pages, max_pages, rope_mode=ROPE_NONE), batch)
    table, lens = cache.block_table.tolist(), [0] * batch
    stack, count = cache.free_pages.tolist(), n_pages
    for step in range(25):
        new = [int(x) for x in g.integers(0, 9, batch)]
        left = (count - 2 * batch) * P
        if sum(new) > left:
            new = [0] * batch
        m = cache.begin(torch.tensor(new, dtype=I32, device=DEV), sum(new) + 1)
        table, lens, _, slots, _, count, refused = plain.page_map(P, n_pages, max_pages, sum(new) + 1, lens, new, stack, count,
                                                                  table)
        assert not refused and m.slots.tolist() == slots and cache.block_table.tolist() == table
        x = torch.randn(sum(new) + 1, 2, 64, device=DEV).half()
        cache.append(0, x, x)
        cache.end()
        done = [int(c > 40 or g.random() < 0.1) for c in lens]
        for b, d in enumerate(done):
            if d:
                for p in range(-(-lens[b] // P)):
                    stack[count] = table[b][p]
                    count += 1
                table[b], lens[b] = [-1] * max_pages, 0
        cache.release(torch.tensor(done, dtype=I32, device=DEV))
        assert cache.block_table.tolist() == table and cache.seq_len.tolist() == lens
        assert cache.free_count.item() == count and cache.free_pages.tolist()[:count] == stack[:count]
        held = [p for r in table for p in r if p >= 0] + stack[:count]
        assert sorted(held) == list(range(n_pages))
    ctx.sync_status()


def test_release_refuses_a_bad_table_whole(ctx):
    ops = Kv8Ops(ctx, Kv8Spec(4, 2, 64, 16, 10, 4))
    t = lambda x: torch.tensor(x, dtype=I32, device=DEV)  # noqa: E731
    table, lens, stack, count = t([[3, 10, -1, -1], [5, -1, -1, -1]]), t([20, 4]), t(list(range(10))), t([4])
    ops.release_pages(t([1, 1]), lens, stack, count, table)
    with pytest.raises(AttnError) as e:
        ctx.sync_status()
    assert e.value.status == A.EINVAL
    assert table.tolist() == [[3, 10, -1, -1], [5, -1, -1, -1]] and lens.tolist() == [20, 4] and count.item() == 4


# ------------------------------------------------------------------------------------------------ append and read

def _append(ctx, w, std_k=1.0, std_v=0.02, spare=0, joined=False):
    k, k64 = w.rows(w.H, std_k)
    v, v64 = w.rows(w.H, std_v)
    if joined:  # K and V as columns of one projection's output
        kv = torch.cat([k, v, v], dim=1).to(DEV)
        kd, vd = kv[:, :w.H], kv[:, w.H:2 * w.H]
    else:
        kd, vd = k.to(DEV), v.to(DEV)
    pools = [w.dev(x) for x in (w.k, w.v, w.ks, w.vs)]
    w.ops.append(kd, vd, w.dev(w.slots), w.dev(w.pos, I32), *pools)
    torch.cuda.synchronize()
    ctx.sync_status()
    k64 = plain.rotate(k64, w.pos, w.theta, w.mode)
    for x, pool, scale, got, got_s in ((k64, w.k, w.ks, pools[0], pools[2]), (v64, w.v, w.vs, pools[1], pools[3])):
        target, s = plain.append(x, w.slots, w.P, pool, scale)
        got, got_s = got.cpu().numpy(), got_s.cpu().numpy().astype(np.float64)
        np.testing.assert_allclose(got_s, s, rtol=2.0 ** -20, atol=0)
        live = ~np.isnan(s)
        far = np.abs(got.astype(np.float64) - target)[live]
        assert far.max() <= 0.5 + 1e-3
    return pools


APPENDS = {
    "one token, fresh page": dict(cached=[0], new=[1]),
    "one token, old rows": dict(cached=[5, 16, 31, 33], new=[1, 1, 1, 1], D=128, H=4),
    "decode batch": dict(cached=list(range(0, 150, 3)), new=[1] * 50, P=32),
    "uneven prompts": dict(cached=[0, 7, 100, 16], new=[70, 0, 33, 129], D=128, P=64),
    "whole pages": dict(cached=[128, 0], new=[256, 128], P=128, D=128),
    "long run on a page": dict(cached=[1], new=[127], P=128, H=1),
    "fp32": dict(cached=[3, 0], new=[40, 17], io=F32, P=32),
    "fp32, d 128": dict(cached=[0, 12], new=[3, 1], io=F32, D=128),
    "rotated pairs": dict(cached=[900, 3], new=[30, 1], mode=ROPE_INTERLEAVED, D=128),
    "rotated halves": dict(cached=[10000, 0], new=[1, 50], mode=ROPE_NEOX, theta=5e5),
    "rotated halves, d 128, fp32": dict(cached=[33], new=[18], mode=ROPE_NEOX, D=128, io=F32),
}


@pytest.mark.parametrize("joined", [False, True])
@pytest.mark.parametrize("case", list(APPENDS))
def test_append(ctx, case, joined):
    _append(ctx, World(ctx, seed=len(case), **APPENDS[case]), joined=joined)


@pytest.mark.parametrize("mode, io", [(ROPE_NONE, F16), (ROPE_INTERLEAVED, F16), (ROPE_NEOX, F32)])
@pytest.mark.parametrize("D, P", [(64, 16), (128, 16), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("new", [[700, 1, 0, 19] + [3] * 130, [2500, 33] + [1] * 150 + [1701]])
def test_append_of_many_rows(ctx, new, D, P, mode, io):
    """From 1024 tokens on, and from 4096: windows over several small pages, two rows to a warp."""
    cached = [(7 * b) % 40 for b in range(len(new))]
    _append(ctx, World(ctx, cached, new, H=3, Hq=3, D=D, P=P, mode=mode, io=io, seed=P))


@pytest.mark.parametrize("std", [1e-6, 100.0])
def test_append_keeps_or_grows_the_scale(ctx, std):
    """Small new rows leave the old rows as they are, large ones bring them to the new scale."""
    w = World(ctx, [9, 20], [1, 5], io=F32, seed=4)
    before = w.k.copy()
    pools = _append(ctx, w, std_k=std)
    page = w.table[0][0]
    old = pools[0][page, :, :9].cpu().numpy()
    assert np.array_equal(old, before[page, :, :9]) == (std < 1)


def test_append_zeros_spares_and_neighbours(ctx):
    """All-zero rows give scale 0 and values 0; slot -1 writes nothing; no other byte of the pools changes."""
    w = World(ctx, [0, 20], [4, 3], seed=5)
    k = torch.zeros(7, w.H, w.D, dtype=torch.float16, device=DEV)
    slots = w.slots.copy()
    slots[5] = -1
    pools = [w.dev(x) for x in (w.k, w.v, w.ks, w.vs)]
    w.ops.append(k, k, w.dev(slots), None, *pools)
    ctx.sync_status()
    fresh = w.table[0][0]
    assert (pools[2][fresh] == 0).all() and (pools[0][fresh, :, :4] == 0).all()
    written = np.zeros(w.k.shape, bool)
    for s in slots[slots >= 0]:
        written[s // w.P, :, s % w.P] = True
    assert np.array_equal(pools[0].cpu().numpy()[~written], w.k[~written])
    assert np.array_equal(pools[3].cpu().numpy()[np.arange(w.n_pages) != fresh], w.vs[np.arange(w.n_pages) != fresh])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("new", [1, 20])
def test_append_of_a_bad_number_marks_its_page_until_begun_anew(ctx, bad, new):
    w = World(ctx, [3], [new], D=128, seed=6)
    k, _ = w.rows(w.H)
    k[0, 1, 77] = bad
    pools = [w.dev(x) for x in (w.k, w.v, w.ks, w.vs)]
    w.ops.append(k.to(DEV), k.to(DEV), w.dev(w.slots), None, *pools)
    ctx.sync_status()
    page = int(w.table[0][0])
    assert torch.isnan(pools[2][page, 1]) and not torch.isnan(pools[2][page, 0])
    k[0, 1, 77] = 1.0
    w.ops.append(k[:1].to(DEV), k[:1].to(DEV), w.dev(np.array([page * 16 + 5])), None, *pools)
    assert torch.isnan(pools[2][page, 1])
    w.ops.append(k[:1].to(DEV), k[:1].to(DEV), w.dev(np.array([page * 16])), None, *pools)
    assert torch.isfinite(pools[2][page]).all()


@pytest.mark.parametrize("D, H, P", [(64, 1, 16), (128, 3, 128)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_read(ctx, D, H, P, dtype):
    w = World(ctx, [50, 300], [1, 1], Hq=H, H=H, D=D, P=P)
    slots = np.concatenate([w.g.permutation(w.n_pages * P)[:97], [-1, 0]])
    got = w.ops.read(w.dev(w.k), w.dev(w.ks), w.dev(slots), dtype).cpu().numpy()
    want = (w.k[slots // P, :, slots % P].astype(np.float32) * w.ks[slots // P][:, :, None])
    want[slots < 0] = 0
    assert np.array_equal(got, want.astype(got.dtype))
    ctx.sync_status()


def test_slots_outside_the_pool_are_skipped_and_reported(ctx):
    w = World(ctx, [4], [2])
    k, _ = w.rows(w.H)
    pools = [w.dev(x) for x in (w.k, w.v, w.ks, w.vs)]
    for bad in (w.n_pages * w.P, -2, 1 << 40):
        w.ops.append(k.to(DEV), k.to(DEV), w.dev(np.array([bad, bad])), None, *pools)
        with pytest.raises(AttnError):
            ctx.sync_status()
        assert (w.ops.read(pools[0], pools[2], w.dev(np.array([bad]))) == 0).all()
        with pytest.raises(AttnError):
            ctx.sync_status()
    assert np.array_equal(pools[0].cpu().numpy(), w.k)


# ------------------------------------------------------------------------------------------------ attention

ATTENDS = {
    "first token": dict(cached=[0], new=[1]),
    "two rows": dict(cached=[1, 0], new=[1, 1], D=128),
    "decode": dict(cached=[15, 16, 17, 300, 1029, 64], new=[1] * 6, D=128, P=64),
    "decode, one head each": dict(cached=[40, 200], new=[1, 1], Hq=3, H=3, D=128, P=32),
    "decode, 3 a group": dict(cached=[99, 5], new=[1, 1], Hq=12, H=4, D=128),
    "decode, 7 a group": dict(cached=[513], new=[1], Hq=14, H=2),
    "decode, 16 a group": dict(cached=[333, 2], new=[1, 1], Hq=32, H=2, D=128, P=128),
    "decode, 20 a group": dict(cached=[100], new=[1], Hq=20, H=1),
    "decode, long": dict(cached=[9000], new=[1], Hq=4, H=1, D=128, P=128),
    "some idle": dict(cached=[50, 60, 70], new=[1, 0, 1]),
    "pair of tokens": dict(cached=[30, 31], new=[2, 1], Hq=8, H=2, P=32),
    "prompts": dict(cached=[0, 100, 37], new=[65, 3, 140], Hq=8, H=2),
    "prompts, d 128": dict(cached=[0, 130, 250], new=[129, 200, 1], Hq=4, H=1, D=128, P=64),
    "prompts, page 128": dict(cached=[127, 1], new=[130, 255], Hq=6, H=2, D=64, P=128),
    "prompt over old rows": dict(cached=[1500], new=[70], Hq=8, H=1, D=128, P=32),
    "given scale": dict(cached=[70], new=[40], scale=0.3),
}


# Which kernel runs, and how the ranges are cut, goes by the bounds that the host gives: with the tight bound these
# small cases take the split-cache kernel, with the loose one several rows a sequence take the tcgen05 kernel.
BOUNDS = [None, 100000]


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("mode", [ROPE_NONE, ROPE_INTERLEAVED, ROPE_NEOX])
@pytest.mark.parametrize("case", list(ATTENDS))
def test_attention(ctx, case, mode, io, max_kv):
    World(ctx, mode=mode, io=io, seed=len(case), **ATTENDS[case]).check(ctx, max_kv=max_kv)


@pytest.mark.parametrize("max_kv", [None, 20000, 60000])
@pytest.mark.parametrize("D, P, mode", [(64, 16, ROPE_NEOX), (128, 128, ROPE_INTERLEAVED), (128, 16, ROPE_NONE)])
def test_attention_in_chunks(ctx, D, P, mode, max_kv):
    """Prompts over long caches: their ranges are cut, by either kernel, and merged."""
    w = World(ctx, [3300, 100, 0, 1500], [90, 40, 33, 1], Hq=8, H=1, D=D, P=P, mode=mode)
    w.check(ctx, max_kv=max_kv)
    w.check(ctx, max_kv=max_kv, prefix=[3000, 139, 40, 0], slopes=[2.0 ** -(h + 1) for h in range(8)])


MASKS = {
    "cap": dict(cap=5.0),
    "bias": dict(slopes=True),
    "prefix": dict(prefix=[0, 20, 90, 1000]),
    "documents": dict(first=True),
    "all": dict(cap=8.0, slopes=True, prefix=[3, 50, 0, 70], first=True),
}


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("D, Hq, H, P", [(64, 8, 2, 16), (128, 8, 8, 64), (128, 32, 4, 32)])
@pytest.mark.parametrize("mask", list(MASKS))
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [5, 33, 0, 150]])
def test_attention_masks(ctx, mask, new, D, Hq, H, P, io, max_kv):
    m = dict(MASKS[mask])
    w = World(ctx, [0, 40, 77, 300], new, Hq=Hq, H=H, D=D, P=P, io=io, cap=m.pop("cap", 0.0), seed=len(mask))
    slopes = [2.0 ** (-8 * (h + 1) / Hq) for h in range(Hq)] if m.get("slopes") else None
    first = None
    if m.get("first"):  # documents of uneven length; every seventh row sees nothing
        first = [int(w.g.integers(0, p + 1)) if t % 7 else p + 1 + 1000 * (t % 2) for t, p in enumerate(w.pos)]
    got = w.check(ctx, std=3.0, slopes=slopes, first=first, prefix=m.get("prefix"), max_kv=max_kv)
    if first is not None and m.get("prefix") is None:
        assert (got[0] == 0).all()


def test_attention_of_capped_and_large_scores(ctx):
    """Scores in the hundreds: the cap saturates, the uncapped softmax is one-hot."""
    for cap in (0.0, 20.0):
        World(ctx, [600], [1], D=128, P=64, io=F32, cap=cap, scale=1.0).check(ctx, std=8.0)


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("cap", [0.5, 3.0, 12.0, 50.0, 1000.0])
@pytest.mark.parametrize("D, P", [(64, 16), (128, 64)])
def test_attention_of_scores_far_below_to_far_above_the_cap(ctx, D, P, cap, max_kv):
    World(ctx, [150, 0, 20], [60, 130, 1], Hq=8, H=2, D=D, P=P, cap=cap, seed=31).check(ctx, max_kv=max_kv)


@pytest.mark.parametrize("max_kv", BOUNDS)
def test_attention_with_uneven_page_scales(ctx, max_kv):
    """V scales from 1e-4 to 10 side by side, and pages of scale zero."""
    w = World(ctx, [500, 90], [1, 30], P=16, D=128)
    w.vs = np.exp(w.g.uniform(np.log(1e-4), np.log(10), w.vs.shape)).astype(np.float32)
    w.ks[::5] = 0
    w.vs[::7] = 0
    w.check(ctx, max_kv=max_kv)
    w.vs[:] = 0
    assert (w.check(ctx, max_kv=max_kv) == 0).all()


@pytest.mark.parametrize("max_kv", BOUNDS)
def test_attention_ignores_what_it_may_not_see(ctx, max_kv):
    """NaN scales on pages in nobody's hands, past the end, before the document, and stale rows on the last page."""
    w = World(ctx, [100, 33], [1, 40], P=16, D=128)
    used = np.zeros(w.n_pages, bool)
    for b, L in enumerate(w.kv_len):
        used[w.table[b][:-(-int(L) // 16)]] = True
    w.ks[~used] = np.nan
    w.vs[~used] = np.nan
    ref = w.check(ctx, max_kv=max_kv)
    assert np.isfinite(ref).all()
    first = [64] + [48 if p >= 48 else 0 for p in w.pos[1:]]
    w.ks[w.table[0][0]] = w.vs[w.table[0][1]] = np.nan  # rows 0..31 of sequence 0, hidden by its document
    w.check(ctx, first=first, max_kv=max_kv)
    w.ks[w.table[1][0]] = np.nan  # rows 0..15 of sequence 1: seen by its first document's rows only
    q, _ = w.rows(w.Hq)
    out = w.attend(q.to(DEV), first=first, max_kv=max_kv).cpu()
    hit = torch.tensor([b == 1 and p < 48 for b, p in zip(np.repeat([0, 1], w.new), w.pos)])
    assert torch.isnan(out[hit]).all() and torch.isfinite(out[~hit]).all()
    w.ks[w.table[1][0]] = 0.01
    w.vs[w.table[1][0]] = np.nan
    out = w.attend(q.to(DEV), first=first, max_kv=max_kv).cpu()
    assert torch.isnan(out[hit]).all() and torch.isfinite(out[~hit]).all()


def test_attention_beyond_32_bit_offsets(ctx):
    """A pool of more than 2^31 bytes with its pages at the far end."""
    P, H, D = 128, 8, 128
    n_pages = (1 << 31) // (P * H * D) + 40
    spec = Kv8Spec(16, H, D, P, n_pages, 4, rope_mode=ROPE_NONE)
    ops = Kv8Ops(ctx, spec)
    pools = [torch.empty(n_pages, H, P, D, dtype=torch.int8, device=DEV) for _ in range(2)]
    scales = [torch.zeros(n_pages, H, device=DEV) for _ in range(2)]
    pages = [n_pages - 1, n_pages - 7]
    table = torch.tensor([pages + [-1, -1]], dtype=I32, device=DEV)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(200, H, D, generator=g).half() for _ in range(2))
    slots = torch.tensor([pages[t // P] * P + t % P for t in range(200)], device=DEV)
    ops.append(k.to(DEV), v.to(DEV), slots, None, pools[0], pools[1], scales[0], scales[1])
    q = torch.randn(200, 16, D, generator=g).half()
    one = lambda x: torch.tensor(x, dtype=I32, device=DEV)  # noqa: E731
    out = ops.attend(q.to(DEV), one([0, 200]), one([200]), table, pools[0], pools[1], scales[0], scales[1], 200, 200)
    last = ops.attend(q[199:].to(DEV), one([0, 1]), one([200]), table, pools[0], pools[1], scales[0], scales[1], 1, 200)
    ctx.sync_status()
    kh, vh = (ops.read(p, s, slots, torch.float32).double().cpu() for p, s in zip(pools, scales))
    assert (kh - k.double()).abs().max() <= k.abs().max() / 127 * 0.51
    x = torch.einsum("thd,jhd->htj", q.double()[:, ::2], kh) / D ** 0.5
    x = x.masked_fill(torch.ones(200, 200).triu(1).bool(), -torch.inf).softmax(-1)
    want = torch.einsum("htj,jhd->thd", x, vh)
    assert (out[:, ::2].double().cpu() - want).abs().max() <= 2e-3
    assert (last[:, ::2].double().cpu() - want[199:]).abs().max() <= 2e-3


@pytest.mark.parametrize("new, loose", [([1, 1], 10 ** 6), ([60, 50], 10 ** 6)])
def test_attention_reports_bad_device_values(ctx, new, loose):
    """A page outside the pool, lengths past the bounds and token counts past the rows: a status, no stray access."""
    w = World(ctx, [40, 100], new, P=16)
    q, _ = w.rows(w.Hq)
    good = w.attend(q.to(DEV), max_kv=loose).clone()

    def refused():
        with pytest.raises(AttnError) as e:
            ctx.sync_status()
        assert e.value.status == A.EINVAL

    table = w.table.copy()
    for bad in (w.n_pages, -1, 2 ** 31 - 1):
        w.table = table.copy()
        w.table[0, 1] = bad
        w.attend(q.to(DEV), max_kv=loose)
        refused()
    w.table = table
    w.attend(q.to(DEV), max_kv=90)
    refused()
    kv, start = w.kv_len.copy(), w.start.copy()
    for i, bad in ((0, 10 ** 6), (1, 0), (1, -5)):
        w.kv_len = kv.copy()
        w.kv_len[i] = bad
        w.attend(q.to(DEV), max_kv=loose)
        refused()
    w.kv_len = kv
    a, b = new
    for bad in ([0, a, a + b + 1], [0, -1, b], [-1, 0, b], [0, a + b, a]):
        w.start = np.array(bad)
        w.attend(q.to(DEV), max_kv=loose)
        refused()
    w.start = start
    assert torch.equal(w.attend(q.to(DEV), max_kv=loose), good)
    ctx.sync_status()


def test_attention_rows_of_a_fused_projection(ctx):
    """q as columns of a wider tensor gives the packed result bit for bit; gaps are not read as rows."""
    for io in (F16, F32):
        for new in ([1, 1], [40, 9]):
            w = World(ctx, [30, 77], new, D=128, io=io, mode=ROPE_INTERLEAVED)
            q, _ = w.rows(w.Hq)
            wide = torch.full((w.T, w.Hq + 5, w.D), float("nan"), dtype=q.dtype)
            wide[:, :w.Hq] = q
            for max_kv in BOUNDS:
                assert torch.equal(w.attend(wide.to(DEV)[:, :w.Hq], max_kv=max_kv), w.attend(q.to(DEV), max_kv=max_kv))


def test_looser_bounds_give_the_same_rows(ctx):
    """max_new and max_kv are bounds: larger ones may split otherwise but stay within the two results' rounding."""
    w = World(ctx, [500, 60], [1, 1], D=128, P=32)
    q, _ = w.rows(w.Hq)
    a = w.attend(q.to(DEV)).float()
    for max_new, max_kv in ((1, 60000), (7, 600), (100, 70000)):
        assert (w.attend(q.to(DEV), max_new=max_new, max_kv=max_kv).float() - a).abs().max() <= 4e-3 * a.abs().max()
    ctx.sync_status()


@pytest.mark.parametrize("new, max_kv", [([1, 1, 1], None), ([70, 9, 300], 30000)])
def test_same_inputs_same_bits(ctx, new, max_kv):
    w = World(ctx, [3000, 900, 77], new, D=128, P=64, Hq=32, H=8)
    q, _ = w.rows(w.Hq)
    first = w.attend(q.to(DEV), max_kv=max_kv).clone()
    for _ in range(10):
        assert torch.equal(w.attend(q.to(DEV), max_kv=max_kv), first)


def test_more_tiles_than_merge_counters(ctx):
    """Too many tiles to merge chunks of: every block takes its whole range, in rounds of 32 blocks of rows a warp. The
    long sequence's rows match the same call on it alone, which is cut into chunks."""
    B, H, long = 1100, 64, 5000
    cached = [long if b == 700 else 3 + b % 20 for b in range(B)]
    w = World(ctx, cached, [1] * B, Hq=H, H=H, D=64, P=16, seed=12)
    q, _ = w.rows(H)
    out = w.attend(q.to(DEV))
    torch.cuda.synchronize()
    ctx.sync_status()
    w.start, w.kv_len, w.table, w.new = np.array([0, 1]), w.kv_len[700:701], w.table[700:701], [1]
    alone = w.attend(q[700:701].to(DEV))
    ctx.sync_status()
    assert (out[700].float() - alone[0].float()).abs().max() <= 2.0 ** -9 * alone.abs().max()


@pytest.mark.parametrize("D, P, mode", [(64, 32, ROPE_NEOX), (128, 64, ROPE_INTERLEAVED), (128, 16, ROPE_NONE)])
def test_whole_tiles_and_the_rest_in_chunks(ctx, D, P, mode):
    """A few more tiles than multiprocessors, ranges alike: most tiles take one block, the last ones (the first 32 rows)
    are cut into chunks. A row's result is that of the row as a single new one over the rows before it."""
    w = World(ctx, [1500], [320], Hq=128, H=8, D=D, P=P, mode=mode, seed=21)
    q, q64 = w.rows(128)
    out = w.attend(q.to(DEV)).double().cpu().numpy()
    ctx.sync_status()
    assert np.isfinite(out).all()
    for i in [0, 15, 16, 31, 32, 47, 200, 319]:
        ref, weight, size = plain.attend(q64[i:i + 1], [0, 1], [1501 + i], w.table, P, w.k, w.v, w.ks, w.vs, w.scale, 0.0,
                                         w.theta, mode)
        ds = size[..., None] * (2.0 ** -19 if mode == ROPE_NONE else 2.0 ** -11)
        tol = 2.0 ** -11 * np.abs(ref) + weight * (2.0 ** -11 + 2.0 ** -16 + 2 * ds) + 1e-7
        assert (np.abs(out[i] - ref[0]) - tol[0]).max() <= 0, i


# ------------------------------------------------------------------------------------------------ together

@pytest.mark.parametrize("D, P, io", [(64, 16, F16), (128, 64, F32)])
def test_steps_of_a_batch(ctx, D, P, io):
    """Prompt, decode and mixed steps through Kv8Cache, two layers, against attention over the unquantised rows (int8
    keeps about 1 % of a row's size) and, exactly bounded, over the rows as the cache holds them."""
    B, Hq, H = 3, 8, 2
    spec = Kv8Spec(Hq, H, D, P, 60, 40 if P == 16 else 12, io, io, rope_mode=ROPE_NEOX)
    cache = Kv8Cache(ctx, spec, B, n_layers=2)
    g = torch.Generator().manual_seed(7)
    full = [[[], []] for _ in range(B)]
    lens = [0] * B
    for new in ([40, 7, 0], [1, 1, 1], [1, 30, 90], [1, 1, 1], [1, 0, 1]):
        T = sum(new)
        m = cache.begin(torch.tensor(new, dtype=I32, device=DEV), T + 2)
        for layer in range(2):
            q, k, v = (torch.randn(T + 2, h, D, generator=g).to(_dt(io)) for h in (Hq, H, H))
            cache.append(layer, k.to(DEV), v.to(DEV))
            out = cache.attend(layer, q.to(DEV), max(new), max(lens) + max(new)).cpu().double().numpy()
            if layer:
                continue
            t = 0
            for b, n in enumerate(new):
                full[b][0].append(plain.rotate(k[t:t + n].double().numpy(), np.arange(lens[b], lens[b] + n), 1e4, ROPE_NEOX))
                full[b][1].append(v[t:t + n].double().numpy())
                kk, vv = (np.concatenate(x) for x in full[b])
                qq = plain.rotate(q[t:t + n].double().numpy(), np.arange(lens[b], lens[b] + n), 1e4, ROPE_NEOX)
                for i in range(n):
                    end = lens[b] + i + 1
                    for h in range(Hq):
                        s = kk[:end, h // (Hq // H)] @ qq[i, h] / D ** 0.5
                        p = np.exp(s - s.max())
                        want = p @ vv[:end, h // (Hq // H)] / p.sum()
                        assert np.abs(out[t + i, h] - want).max() < 0.12
                t += n
        cache.end()
        lens = [c + n for c, n in zip(lens, new)]
        assert cache.seq_len.tolist() == lens
    ctx.sync_status()
    with pytest.raises(AttnError):
        cache.end()


def test_on_another_stream_and_in_a_graph(ctx):
    """A captured decode step (map, append, attend) with spare tokens, replayed over changing inputs."""
    B, H, Hq, D, P = 4, 2, 8, 64, 16
    spec = Kv8Spec(Hq, H, D, P, 50, 8, rope_mode=ROPE_INTERLEAVED)
    side = torch.cuda.Stream()
    g = torch.Generator().manual_seed(9)
    eager, captured = (Kv8Cache(ctx, spec, B, stream=s) for s in (None, side))
    ones = torch.ones(B, dtype=I32, device=DEV)
    q, k, v = (torch.zeros(B, h, D, dtype=torch.float16, device=DEV) for h in (Hq, H, H))
    ops, c = captured.ops, captured
    from aihost_b200.kv8 import StepMap

    m = StepMap(c.seq_len, torch.zeros(B + 1, dtype=I32, device=DEV), torch.zeros(B + 3, dtype=torch.int64, device=DEV),
                torch.zeros(B + 3, dtype=I32, device=DEV), c.free_count)
    out = torch.zeros(B, Hq, D, dtype=torch.float16, device=DEV)
    ops.attend(q, torch.zeros(B + 1, dtype=I32, device=DEV), c.seq_len, c.block_table, c.k[0], c.v[0], c.k_scale[0],
               c.v_scale[0], 1, 128, out=out)  # sizes the scratch before the capture
    torch.cuda.synchronize()

    def step():
        ops.map_pages(c.seq_len, ones, c.free_pages, c.free_count, c.block_table, B + 3, into=m)
        ops.append(k, v, m.slots, m.positions, c.k[0], c.v[0], c.k_scale[0], c.v_scale[0])
        ops.attend(q, m.row_start, m.kv_len, c.block_table, c.k[0], c.v[0], c.k_scale[0], c.v_scale[0], 1, 128, out=out)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for _ in range(40):
        for x, h in ((q, Hq), (k, H), (v, H)):
            x.copy_(torch.randn(B, h, D, generator=g).half())
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager.begin(ones, B)
        eager.append(0, k, v)
        want = eager.attend(0, q, 1, 128)
        eager.end()
        assert torch.equal(out, want)
    assert c.seq_len.tolist() == [40] * B and eager.seq_len.tolist() == [40] * B
    ctx.sync_status()


def test_split_attention_in_a_graph(ctx):
    """A captured call whose chunks are merged by the last block, replayed over changing queries, between eager calls."""
    w = World(ctx, [3000, 40, 0], [1, 1, 1], D=128, P=64)
    q = torch.zeros(w.T, w.Hq, w.D, dtype=torch.float16, device=DEV)
    args = [w.dev(x, I32) for x in (w.start, w.kv_len, w.table)] + [w.dev(x) for x in (w.k, w.v, w.ks, w.vs)]
    out, side = torch.empty_like(q), torch.cuda.Stream()
    w.ops.attend(q, *args, 1, 3001, out=out)
    torch.cuda.synchronize()
    graph, ops = torch.cuda.CUDAGraph(), Kv8Ops(ctx, w.spec, side)
    with torch.cuda.graph(graph, stream=side):
        ops.attend(q, *args, 1, 3001, out=out)
    for _ in range(5):
        q.copy_(w.rows(w.Hq)[0])
        torch.cuda.synchronize()
        for _ in range(3):
            out.zero_()
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w.ops.attend(q, *args, 1, 3001))
        torch.cuda.synchronize()
    ctx.sync_status()


def test_arguments_are_checked_in_python_too(ctx):
    w = World(ctx, [20], [1])
    q, _ = w.rows(w.Hq)
    q = q.to(DEV)
    for bad in (q.float(), q.cpu(), q[:, :4], q.transpose(1, 2)):
        with pytest.raises(AttnError) as e:
            w.attend(bad)
        assert e.value.status == A.EINVAL
    with pytest.raises(AttnError):
        w.ops.read(w.dev(w.k)[1:], w.dev(w.ks), w.dev(w.slots))
    with pytest.raises(AttnError):
        w.ops.append(q[:, :2], q[:, 1:4], w.dev(w.slots), None, w.dev(w.k), w.dev(w.v), w.dev(w.ks), w.dev(w.vs))
    with pytest.raises(AttnError) as e:
        Kv8Ops(ctx, dataclasses.replace(w.spec, head_dim=96)).read(w.dev(w.k), w.dev(w.ks), w.dev(w.slots))
    assert e.value.status in (A.EINVAL, A.EUNSUPPORTED)


def test_server_loop(ctx):
    """The example: every page comes back, and int8 rows stay near the unquantised ones (a page's rounding step is its
    largest value / 127, about 4 / 127 for normal rows; half of it in V, and as much again through the scores)."""
    from aihost_b200 import serve_kv8

    r = serve_kv8.main(["--batch", "5", "--requests", "11", "--layers", "2", "--prompt", "150", "--answer", "12"])
    assert r["free"] == r["pages"] and r["worst"] < 0.1
