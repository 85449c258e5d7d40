"""The 4-bit paged cache on the GPU against plain forms (tests/kv4_plain.py).

  append     codes and ranges are defined to the bit
  attention  fp16: the output's rounding 2^-11 |o|; P's rounding 2^-11 of sum p |v - low - 8 step|, and fp32 sums; the score's error ds shifts p by up to 2 ds, ds = 2^-19 of sum |q| kmax, kmax =
             max(|low|, |low + 15 step|) of the row (codes and low enter apart); for a rotated q 2^-18, the rotation's
             fp32 arithmetic
             fp32: pairs of fp16 hold 22 bits; ex2.approx and fp32 sums 2^-18 of sum p vmax and 2^-19 of sum |q| kmax
"""
import numpy as np
import pytest
import torch

import aihost_b200 as A
import kv4_plain as plain4
import kv8_plain as plain
from aihost_b200 import F16, F32, KV8_SPLIT_CACHE, KV8_TENSOR, ROPE_INTERLEAVED, ROPE_NEOX, ROPE_NONE, AttnError
from aihost_b200.kv4 import Kv4Cache, Kv4Ops, Kv4Spec
from aihost_b200.ops import Context
from test_gpu_kv8 import ATTENDS, BOUNDS, DEV, I32, MASKS, World
from test_gpu_kv8_cold import cold_calls

pytestmark = pytest.mark.gpu


class World4(World):
    """A 4-bit pool with scattered pages, filled with noise, and a step of new rows on top."""

    def __init__(self, ctx, cached, new, **kw):
        super().__init__(ctx, cached, new, **kw)
        s = self.spec
        self.spec = Kv4Spec(**{f: getattr(s, f) for f in s.__dataclass_fields__})
        self.ops = Kv4Ops(ctx, self.spec)
        shape = (self.n_pages, self.H, self.P)
        self.k, self.v = (self.g.integers(0, 256, (*shape, self.D // 2)).astype(np.uint8) for _ in range(2))
        self.ks, self.vs = (self._ranges(shape) for _ in range(2))

    def _ranges(self, shape):
        step = self.g.uniform(0.05, 0.4, shape)
        return np.stack([self.g.normal(0, 0.5, shape) - 7.5 * step, step], -1).astype(np.float16)

    def reference(self, q64, prefix=None, first=None, slopes=None):
        """(out, what P's rounding goes by, sum p vmax, the largest scale sum |q| kmax), of every element and row."""
        one = np.ones(self.ks.shape[:2])
        k, v = (plain4.values(p, r, np.float64) for p, r in ((self.k, self.ks), (self.v, self.vs)))
        rest = (q64, self.start, self.kv_len, self.table, self.P)
        more = (one, one, self.scale, self.cap, self.theta, self.mode, prefix, first, None if slopes is None else np.float32(slopes))
        out = plain.attend(*rest, k, v, *more)[0]
        low, step = (self.vs[..., i:i + 1].astype(np.float64) for i in (0, 1))
        off = plain.attend(*rest, k, v - low - 8 * step, *more)[1]
        top = lambda r: np.maximum(abs(r[..., :1]), abs(r[..., :1] + 15 * r[..., 1:])).repeat(self.D, -1)  # noqa: E731
        most = plain.attend(*rest, k, top(self.vs.astype(np.float64)), *more)[1]
        size = plain.attend(*rest, top(self.ks.astype(np.float64)), v, *more)[2]
        return out, off, most, size

    def check(self, ctx, std=1.0, prefix=None, first=None, slopes=None, **kw):
        q, q64 = self.rows(self.Hq, std)
        out = self.attend(q.to(DEV), prefix=prefix, first=first, slopes=slopes, **kw)
        torch.cuda.synchronize()
        ctx.sync_status()
        ref, off, most, size = self.reference(q64, prefix, first, slopes)
        got = out.double().cpu().numpy()
        ds = size[..., None] * (2.0 ** -19 if self.mode == ROPE_NONE or self.io == F32 else 2.0 ** -18)
        if self.io == F16:
            tol = 2.0 ** -11 * np.abs(ref) + off * 2.0 ** -11 + most * (2.0 ** -16 + 2 * ds) + 1e-7
        else:
            tol = most * (2.0 ** -18 + 2 * ds) + 1e-9
        over = np.abs(got - ref) - tol
        bad = np.argwhere((over > 0).any(-1))  # (row, head)
        assert np.isfinite(got).all() and not len(bad), (over.max(), len(bad), bad[:5].tolist(), bad[-1].tolist())
        return got

    def pools(self):
        return [self.dev(x) for x in (self.k, self.v, self.ks, self.vs)]


# ------------------------------------------------------------------------------------------------ append and read

def _expect(w, k, v, slots=None):
    """The pools and ranges that appending k, v (as torch rows) has to give."""
    slots = w.slots if slots is None else slots
    want = [x.copy() for x in (w.k, w.v, w.ks, w.vs)]
    k32 = plain4.rotate32(k.float().numpy(), w.pos, w.theta, w.mode)
    on = slots >= 0
    at = (slots[on] // w.P, slice(None), slots[on] % w.P)
    for i, x in enumerate((k32, v.float().numpy())):
        codes, low, step = plain4.quantise(x[on])
        want[i][at] = plain4.pack(codes)
        want[2 + i][at] = np.stack([low, step], -1)
    return want


def _append(ctx, w, k, v, slots=None):
    pools = w.pools()
    slots = w.slots if slots is None else slots
    w.ops.append(k.to(DEV), v.to(DEV), w.dev(slots), w.dev(w.pos, I32) if w.mode != ROPE_NONE else None, *pools)
    ctx.sync_status()
    for got, want in zip(pools, _expect(w, k, v, slots)):
        assert np.array_equal(got.cpu().numpy(), want, equal_nan=want.dtype == np.float16)
    return pools


@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("mode", [ROPE_NONE, ROPE_INTERLEAVED, ROPE_NEOX])
@pytest.mark.parametrize("D, H, P, cached, new", [
    (64, 1, 16, [0], [1]), (128, 1, 16, [15, 16, 17, 0], [1, 1, 1, 1]), (64, 3, 32, [3, 0, 40], [7, 0, 33]),
    (128, 5, 128, [100, 5], [60, 130]), (64, 9, 64, [1], [1500]), (128, 8, 64, [70000, 2], [700, 400])])
def test_append_to_the_bit(ctx, D, H, P, cached, new, mode, io):
    w = World4(ctx, cached, new, Hq=H, H=H, D=D, P=P, mode=mode, io=io, theta=5e5, seed=D + P)
    _append(ctx, w, w.rows(H)[0], w.rows(H, std=0.3)[0])


@pytest.mark.parametrize("io", [F16, F32])
def test_append_of_rows_of_every_size(ctx, io):
    """Rows alike, zeros, from fp16's smallest numbers to its largest, and fp32 rows beyond: to the bit, NaN where the range
    passes fp16's."""
    w = World4(ctx, [0], [64], Hq=2, H=2, D=64, io=io, seed=3)
    k, v = w.rows(2)[0], w.rows(2)[0]
    size = torch.logspace(-9, 5.3 if io == F32 else 4.2, 64)[:, None, None]
    k, v = (k.float() * size).to(k.dtype), (v.float() * size.flip(0) + size).to(v.dtype)
    k[3], v[5], k[7] = 0.0, -2.5, 65504.0
    pools = _append(ctx, w, k, v)
    assert torch.isnan(pools[2]).any() == (io == F32)
    k64 = plain4.values(pools[0].cpu().numpy(), pools[2].cpu().numpy(), np.float64)[w.slots // w.P, :, w.slots % w.P]
    x = k.double().numpy()
    fine = np.isfinite(k64).all(-1)
    spread = (x.max(-1) - x.min(-1))[..., None]
    # half a step, that rounded to fp16 once, low rounded to fp16 once, the step at least 2^-24
    tol = spread / 30 * (1 + 2.0 ** -10) + spread * 2.0 ** -11 + np.abs(x).max(-1, keepdims=True) * 2.0 ** -11 + 2.0 ** -24 * 16
    assert (np.abs(k64 - x) <= tol)[fine].all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("io", [F16, F32])
def test_append_of_a_bad_number_marks_its_row_alone(ctx, bad, io):
    w = World4(ctx, [3], [20], D=128, io=io, seed=6)
    k, v = w.rows(w.H)[0], w.rows(w.H)[0]
    k[4, 1, 77] = v[9, 0, 3] = bad
    pools = _append(ctx, w, k, v)
    page, row = divmod(int(w.slots[4]), w.P)
    assert torch.isnan(pools[2][page, 1, row]).all() and torch.isfinite(pools[2][page, 0]).all()


def test_append_skips_spares_takes_any_order_and_leaves_other_rows(ctx):
    w = World4(ctx, [0, 20], [9, 30], D=64, seed=5)
    slots = w.slots.copy()
    slots[[5, 17]] = -1
    order = w.g.permutation(w.T)
    k, v = w.rows(w.H)[0], w.rows(w.H)[0]
    _append(ctx, w, k, v, slots)
    w.slots = w.slots[order]
    _append(ctx, w, k, v, slots[order])


@pytest.mark.parametrize("H, D, dtype", [(2, 64, torch.float16), (3, 128, torch.float32)])
def test_append_of_a_fused_projection(ctx, H, D, dtype):
    """k and v as columns of one tensor: the same as packed."""
    w = World4(ctx, [7], [33], Hq=H, H=H, D=D, io=F16 if dtype == torch.float16 else F32, mode=ROPE_NEOX, seed=8)
    x = torch.randn(33, 3 * H, D, generator=torch.Generator().manual_seed(2)).to(dtype)
    pools = w.pools()
    y = x.to(DEV)
    w.ops.append(y[:, H:2 * H], y[:, 2 * H:], w.dev(w.slots), w.dev(w.pos, I32), *pools)
    ctx.sync_status()
    for got, want in zip(pools, _expect(w, x[:, H:2 * H], x[:, 2 * H:])):
        assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("D, H, P", [(64, 1, 16), (128, 3, 128), (128, 40, 32)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_read(ctx, D, H, P, dtype):
    w = World4(ctx, [50, 300], [1, 1], Hq=H, H=H, D=D, P=P)
    slots = np.concatenate([w.g.permutation(w.n_pages * P)[:97], [-1, 0]])
    got = w.ops.read(w.dev(w.k), w.dev(w.ks), w.dev(slots), dtype).cpu().numpy()
    want = plain4.values(w.k[slots // P, :, slots % P], w.ks[slots // P, :, slots % P])
    want[slots < 0] = 0
    assert np.array_equal(got, want.astype(got.dtype))
    ctx.sync_status()


def test_slots_outside_the_pool_are_skipped_and_reported(ctx):
    w = World4(ctx, [4], [2])
    k, _ = w.rows(w.H)
    pools = w.pools()
    for bad in (w.n_pages * w.P, -2, 1 << 40):
        w.ops.append(k.to(DEV), k.to(DEV), w.dev(np.array([bad, bad])), None, *pools)
        with pytest.raises(AttnError):
            ctx.sync_status()
        assert (w.ops.read(pools[0], pools[2], w.dev(np.array([bad]))) == 0).all()
        with pytest.raises(AttnError):
            ctx.sync_status()
    for got, was in zip(pools, (w.k, w.v, w.ks, w.vs)):
        assert np.array_equal(got.cpu().numpy(), was)


# ------------------------------------------------------------------------------------------------ attention

@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("mode", [ROPE_NONE, ROPE_INTERLEAVED, ROPE_NEOX])
@pytest.mark.parametrize("case", list(ATTENDS))
def test_attention(ctx, case, mode, io, max_kv):
    World4(ctx, mode=mode, io=io, seed=len(case), **ATTENDS[case]).check(ctx, max_kv=max_kv)


@pytest.mark.parametrize("max_kv", [None, 20000, 60000])
@pytest.mark.parametrize("D, P, mode", [(64, 16, ROPE_NEOX), (128, 128, ROPE_INTERLEAVED), (128, 16, ROPE_NONE)])
def test_attention_in_chunks(ctx, D, P, mode, max_kv):
    w = World4(ctx, [3300, 100, 0, 1500], [90, 40, 33, 1], Hq=8, H=1, D=D, P=P, mode=mode)
    w.check(ctx, max_kv=max_kv)
    w.check(ctx, max_kv=max_kv, prefix=[3000, 139, 40, 0], slopes=[2.0 ** -(h + 1) for h in range(8)])


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("D, Hq, H, P", [(64, 8, 2, 16), (128, 8, 8, 64), (128, 32, 4, 32)])
@pytest.mark.parametrize("mask", list(MASKS))
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [5, 33, 0, 150]])
def test_attention_masks(ctx, mask, new, D, Hq, H, P, io, max_kv):
    m = dict(MASKS[mask])
    w = World4(ctx, [0, 40, 77, 300], new, Hq=Hq, H=H, D=D, P=P, io=io, cap=m.pop("cap", 0.0), seed=len(mask))
    slopes = [2.0 ** (-8 * (h + 1) / Hq) for h in range(Hq)] if m.get("slopes") else None
    first = None
    if m.get("first"):  # documents of uneven length; every seventh row sees nothing
        first = [int(w.g.integers(0, p + 1)) if t % 7 else p + 1 + 1000 * (t % 2) for t, p in enumerate(w.pos)]
    got = w.check(ctx, std=3.0, slopes=slopes, first=first, prefix=m.get("prefix"), max_kv=max_kv)
    if first is not None and m.get("prefix") is None:
        assert (got[0] == 0).all()


@pytest.mark.parametrize("mode", [ROPE_INTERLEAVED, ROPE_NEOX])
@pytest.mark.parametrize("G, new", [(1, [4, 2, 0, 3]), (2, [2, 1, 2, 0]), (3, [1, 1, 0, 1]), (4, [1, 1, 1, 1]), (1, [5, 8, 1, 2])])
@pytest.mark.parametrize("D, P", [(64, 16), (128, 64)])
def test_up_to_four_rotated_rows(ctx, D, P, G, new, mode):
    """Whose two parts share a product, and those just past four, with every mask."""
    w = World4(ctx, [700, 0, 33, 2100], new, Hq=2 * G, H=2, D=D, P=P, mode=mode, theta=5e5, seed=G + D)
    w.check(ctx, std=2.0)
    first = [int(w.g.integers(0, p + 1)) for p in w.pos]
    w.check(ctx, std=2.0, first=first, slopes=[2.0 ** -(h + 1) for h in range(2 * G)])
    w.check(ctx, std=2.0, prefix=[705, 1, 35, 0])


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("io", [F16, F32])
def test_the_largest_steps(ctx, io, max_kv):
    """Steps that an append does not make, up to fp16's largest, with values that stay in its range."""
    w = World4(ctx, [90, 20], [40, 3], P=16, D=128, io=io, seed=5)
    w.vs[...] = np.float16([-65504.0, 65504.0])
    w.v = w.v & 0x33 & ~(w.v >> 1 & 0x11)  # codes 0, 1 and 2
    w.check(ctx, max_kv=max_kv)


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("cap", [1e-25, 0.5, 12.0, 1000.0, 1e35])
@pytest.mark.parametrize("D, P, io", [(64, 16, F16), (128, 64, F16), (128, 32, F32)])
def test_attention_of_scores_far_below_to_far_above_the_cap(ctx, D, P, cap, io, max_kv):
    World4(ctx, [150, 0, 20], [60, 130, 1], Hq=8, H=2, D=D, P=P, cap=cap, io=io, seed=31).check(ctx, max_kv=max_kv)


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("low, high", [(2.0 ** -24, 2.0 ** -20), (1e-4, 10.0), (2.0 ** -24, 4000.0)])
def test_attention_with_uneven_steps(ctx, io, low, high, max_kv):
    """Steps far apart side by side, and rows whose step is zero (their low alone)."""
    w = World4(ctx, [500, 90, 40], [1, 30, 3], P=16, D=128, io=io, seed=12)
    step = np.exp(w.g.uniform(np.log(low), np.log(high), w.vs.shape[:-1])).astype(np.float16)
    step[:, :, ::5] = 0
    w.vs = np.stack([-7 * step.astype(np.float32), step], -1).astype(np.float16)
    w.ks[:, :, ::7, 1] = 0
    w.check(ctx, max_kv=max_kv)


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("io", [F16, F32])
@pytest.mark.parametrize("D, P", [(64, 16), (128, 128)])
def test_documents_whose_values_differ_in_size(ctx, D, P, io, max_kv):
    """A document of small values beside one of large ones, ending inside a page: its rows keep their weights' bits."""
    w = World4(ctx, [200, 77], [1, 60], P=P, D=D, io=io, seed=14)
    for b, end in ((0, 90), (1, 83)):
        for t in range(int(w.kv_len[b])):
            page, row = w.table[b][t // P], t % P
            step = 2.0 ** -18 if t >= end else 1000.0
            w.vs[page, :, row] = np.float16([-6 * step, step])
    first = [90] + [83 if p >= 83 else 0 for p in w.pos[1:]]
    q, q64 = w.rows(w.Hq)
    out = w.attend(q.to(DEV), first=first, max_kv=max_kv).double().cpu().numpy()
    ctx.sync_status()
    ref, off, most, size = w.reference(q64, first=first)
    tol = 2.0 ** -11 * np.abs(ref) + off * 2.0 ** -11 + most * (2.0 ** -16 + 2.0 ** -18 * size[..., None]) + (2.0 ** -25 if io == F16 else 1e-12)
    assert (np.abs(out - ref) <= tol).all()


@pytest.mark.parametrize("std", [1e-6, 300.0, 1e30])
@pytest.mark.parametrize("mode", [ROPE_NONE, ROPE_NEOX])
def test_fp32_queries_of_any_size(ctx, std, mode):
    w = World4(ctx, [300, 40], [1, 5], D=128, P=32, io=F32, mode=mode, scale=1.0 / std, seed=9)
    q, q64 = w.rows(w.Hq, std)
    got = w.attend(q.to(DEV)).double().cpu().numpy()
    ref, _, most, size = w.reference(q64)
    assert (np.abs(got - ref) <= most * (2.0 ** -18 + 2.0 ** -18 * size[..., None]) + 1e-9).all()


@pytest.mark.parametrize("max_kv", BOUNDS)
@pytest.mark.parametrize("io", [F16, F32])
def test_attention_ignores_what_it_may_not_see(ctx, io, max_kv):
    """NaN ranges on pages in nobody's hands, past the end, before the document, and stale rows on the last page."""
    w = World4(ctx, [100, 33], [1, 40], P=16, D=128, io=io)
    used = np.zeros((w.n_pages, w.P), bool)
    for b, L in enumerate(w.kv_len):
        t = np.arange(int(L))
        used[w.table[b][t // 16], t % 16] = True
    for r in (w.ks, w.vs):
        r.transpose(0, 2, 1, 3)[~used] = np.nan
    ref = w.check(ctx, max_kv=max_kv)
    assert np.isfinite(ref).all()
    first = [64] + [48 if p >= 48 else 0 for p in w.pos[1:]]
    w.ks[w.table[0][0]] = w.vs[w.table[0][1]] = np.nan  # rows 0..31 of sequence 0, hidden by its document
    w.check(ctx, first=first, max_kv=max_kv)
    hit = torch.tensor([b == 1 and p < 48 for b, p in zip(np.repeat([0, 1], w.new), w.pos)])
    q, _ = w.rows(w.Hq)
    keep = [x.copy() for x in (w.ks, w.vs)]
    for which, col, bad in (("ks", 0, np.nan), ("ks", 1, np.nan), ("vs", 0, np.nan), ("vs", 1, np.nan), ("vs", 1, np.inf)):
        w.ks, w.vs = (x.copy() for x in keep)
        getattr(w, which)[w.table[1][0], :, 3, col] = bad  # row 3 of sequence 1: seen by its first document's rows only
        out = w.attend(q.to(DEV), first=first, max_kv=max_kv).cpu()
        assert torch.isnan(out[hit]).all() and torch.isfinite(out[~hit]).all()


def test_attention_beyond_32_bit_offsets(ctx):
    """A pool of more than 2^31 bytes with its pages at the far end."""
    P, H, D = 128, 8, 128
    n_pages = (1 << 31) // (P * H * D // 2) + 40
    ops = Kv4Ops(ctx, Kv4Spec(16, H, D, P, n_pages, 4, rope_mode=ROPE_NONE))
    pools = [torch.empty(n_pages, H, P, D // 2, dtype=torch.uint8, device=DEV) for _ in range(2)]
    ranges = [torch.zeros(n_pages, H, P, 2, dtype=torch.float16, device=DEV) for _ in range(2)]
    pages = [n_pages - 1, n_pages - 7]
    table = torch.tensor([pages + [-1, -1]], dtype=I32, device=DEV)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(200, H, D, generator=g).half() for _ in range(2))
    slots = torch.tensor([pages[t // P] * P + t % P for t in range(200)], device=DEV)
    ops.append(k.to(DEV), v.to(DEV), slots, None, *pools, *ranges)
    q = torch.randn(200, 16, D, generator=g).half()
    one = lambda x: torch.tensor(x, dtype=I32, device=DEV)  # noqa: E731
    out = ops.attend(q.to(DEV), one([0, 200]), one([200]), table, *pools, *ranges, 200, 200)
    last = ops.attend(q[199:].to(DEV), one([0, 1]), one([200]), table, *pools, *ranges, 1, 200)
    ctx.sync_status()
    kh, vh = (ops.read(p, s, slots, torch.float32).double().cpu() for p, s in zip(pools, ranges))
    spread = k.double().amax(-1, keepdim=True) - k.double().amin(-1, keepdim=True)
    assert ((kh - k.double()).abs() <= spread * (1 / 30 + 2.0 ** -10)).all()
    x = torch.einsum("thd,jhd->htj", q.double()[:, ::2], kh) / D ** 0.5
    x = x.masked_fill(torch.ones(200, 200).triu(1).bool(), -torch.inf).softmax(-1)
    want = torch.einsum("htj,jhd->thd", x, vh)
    assert (out[:, ::2].double().cpu() - want).abs().max() <= 2e-3
    assert (last[:, ::2].double().cpu() - want[199:]).abs().max() <= 2e-3


@pytest.mark.parametrize("new, loose", [([1, 1], False), ([30, 3], False), ([30, 3], True)])
def test_attention_reports_bad_device_values(ctx, new, loose):
    """Pages outside the pool and lengths out of bounds are not followed: a status, and the other sequence's rows as they
    are."""
    bound = 100000 if loose else None
    w = World4(ctx, [40, 50], new, P=16, D=128, seed=2)
    q, q64 = w.rows(w.Hq)
    want = w.reference(q64)[0]
    t1 = new[0]
    for change in ("page", "length", "start"):
        v = World4(ctx, [40, 50], new, P=16, D=128, seed=2)
        if change == "page":
            v.table[0, 1] = v.n_pages
        elif change == "length":
            v.kv_len = v.kv_len.copy()
            v.kv_len[0] = 1 << 30
        else:
            v.kv_len = v.kv_len.copy()
            v.kv_len[0] = new[0] - 1
        out = v.attend(q.to(DEV), max_kv=bound or 100).double().cpu().numpy()
        with pytest.raises(AttnError):
            ctx.sync_status()
        assert np.abs(out[t1:] - want[t1:]).max() < 2e-2
    ctx.sync_status()


@pytest.mark.parametrize("new, max_kv", [([1, 1], None), ([70, 40], None), ([70, 40], 100000)])
def test_same_inputs_same_bits_and_rows_of_no_sequence_stay(ctx, new, max_kv):
    w = World4(ctx, [700, 90], new, D=128, P=64, mode=ROPE_INTERLEAVED)
    q = torch.cat([w.rows(w.Hq)[0], torch.randn(9, w.Hq, w.D).half()]).to(DEV)
    outs = []
    for _ in range(3):
        out = torch.full_like(q, 7.0)
        outs.append(w.ops.attend(q, w.dev(w.start, I32), w.dev(w.kv_len, I32), w.dev(w.table, I32), *w.pools(), max(new),
                                 max_kv or int(w.kv_len.max()), out=out))
    ctx.sync_status()
    assert all(torch.equal(x, outs[0]) for x in outs) and (outs[0][w.T:] == 7.0).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mode", [ROPE_NONE, ROPE_NEOX])
@pytest.mark.parametrize("shape", [dict(cached=[700, 1], new=[64, 255], Hq=8), dict(cached=[127, 1], new=[130, 255], Hq=6)])
def test_calls_from_cold_caches(ctx, D, mode, shape):
    w = World4(ctx, H=2, D=D, P=128, mode=mode, seed=17, **shape)
    assert cold_calls(w, (w.k, w.v, w.ks, w.vs), 1000) == 0
    ctx.sync_status()


def test_attention_rows_of_a_fused_projection(ctx):
    w = World4(ctx, [60, 9], [1, 20], D=128, P=32, mode=ROPE_NEOX)
    qkv = torch.randn(w.T, w.Hq + 4, w.D, generator=torch.Generator().manual_seed(3)).half().to(DEV)
    assert torch.equal(w.attend(qkv[:, :w.Hq]), w.attend(qkv[:, :w.Hq].contiguous()))


def test_more_tiles_than_merge_counters(ctx):
    """More (tile, head) units than can be merged: one chunk each."""
    n = 70000
    ops = Kv4Ops(ctx, Kv4Spec(1, 1, 64, 16, 40, 40, rope_mode=ROPE_NONE))
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(600, 1, 64, generator=g).half().to(DEV) for _ in range(2))
    pools = [torch.zeros(40, 1, 16, 32, dtype=torch.uint8, device=DEV) for _ in range(2)]
    ranges = [torch.zeros(40, 1, 16, 2, dtype=torch.float16, device=DEV) for _ in range(2)]
    ops.append(k, v, torch.arange(600, device=DEV), None, *pools, *ranges)
    q = torch.randn(1, 1, 64, generator=g).half().to(DEV)
    table = torch.arange(40, dtype=I32, device=DEV)
    out = ops.attend(q.expand(n, 1, 64).contiguous(), torch.arange(n + 1, dtype=I32, device=DEV), torch.full((n,), 600, dtype=I32, device=DEV),
                     table.expand(n, 40).contiguous(), *pools, *ranges, 1, 600)
    ctx.sync_status()
    kh, vh = (ops.read(p, r, torch.arange(600, device=DEV), torch.float32).double() for p, r in zip(pools, ranges))
    want = torch.softmax((kh[:, 0] @ q[0, 0].double()) / 8, 0) @ vh[:, 0]
    assert (out.double() - want).abs().max() <= 2e-3 and (out == out[0]).all()


# ------------------------------------------------------------------------------------------------ steps, graphs, streams

@pytest.mark.parametrize("D, P, io", [(64, 16, F32), (128, 64, F16)])
def test_steps_of_a_batch(ctx, D, P, io):
    """Requests come and go over Kv4Cache: every step's attention against 64-bit attention over the values that the cache
    holds."""
    B, H, Hq, layers = 4, 2, 6, 2
    dt = torch.float16 if io == F16 else torch.float32
    spec = Kv4Spec(Hq, H, D, P, n_pages=B * 8, max_pages=-(-200 // P) + 1, io_dtype=io, out_dtype=io, rope_mode=ROPE_NEOX)
    cache = Kv4Cache(ctx, spec, B, layers)
    rng, g = np.random.default_rng(0), torch.Generator().manual_seed(0)
    lens, held = [0] * B, [[np.zeros((0, H, D))] * 2 for _ in range(B)]
    for step in range(8):
        new = [int(rng.integers(0, 20 if step % 3 == 0 else 3)) for _ in range(B)]
        T = sum(new)
        m = cache.begin(torch.tensor(new, dtype=I32, device=DEV), T + 2)
        q, k, v = (torch.randn(T + 2, h, D, generator=g).to(dt) for h in (Hq, H, H))
        for layer in range(layers):
            cache.append(layer, k.to(DEV), v.to(DEV))
            out = cache.attend(layer, q.to(DEV), max(max(new), 1), 200)
        cache.end()
        ctx.sync_status()
        slots = m.slots[:T]
        kh, vh = (cache.ops.read(p[1], r[1], slots, torch.float32).double().cpu().numpy() for p, r in ((cache.k, cache.k_range), (cache.v, cache.v_range)))
        at = 0
        for b, n in enumerate(new):
            held[b] = [np.concatenate([old, x[at:at + n]]) for old, x in zip(held[b], (kh, vh))]
            if n:
                K, V = held[b]
                qb = plain.rotate(q[at:at + n].double().numpy(), np.arange(lens[b], lens[b] + n), 1e4, ROPE_NEOX)
                for h in range(Hq):
                    s = qb[:, h] @ K[:, h // 3].T / D ** 0.5
                    s[np.arange(lens[b] + n)[None, :] > lens[b] + np.arange(n)[:, None]] = -np.inf
                    w = np.exp(s - s.max(-1, keepdims=True))
                    w /= w.sum(-1, keepdims=True)
                    assert np.abs(out[at:at + n, h].double().cpu().numpy() - w @ V[:, h // 3]).max() < (4e-3 if io == F16 else 4e-5)
            lens[b] += n
            at += n
        done = [int(rng.random() < 0.25 or lens[b] > 150) for b in range(B)]
        cache.release(torch.tensor(done, dtype=I32, device=DEV))
        for b in range(B):
            if done[b]:
                lens[b], held[b] = 0, [np.zeros((0, H, D))] * 2
    assert cache.free_count.item() == spec.n_pages - sum(-(-x // P) for x in lens)


@pytest.mark.parametrize("new, max_kv", [([1, 1, 1], 3001), ([64, 3, 40], 20000)])
def test_in_a_graph_on_a_stream_and_after_the_scratch_has_grown(new, max_kv):
    """Append and attention captured on a side stream, replayed with new rows after the context's scratch has grown."""
    with Context(0) as own:
        w = World4(own, [2900, 40, 700], new, D=128, P=64, mode=ROPE_INTERLEAVED)
        pools, side = w.pools(), torch.cuda.Stream()
        q, k, v = (w.rows(h)[0].to(DEV) for h in (w.Hq, w.H, w.H))
        slots, pos, start, lens, table = (w.dev(w.slots), *(w.dev(x, I32) for x in (w.pos, w.start, w.kv_len, w.table)))
        out = torch.empty_like(q)

        def step(ops):
            ops.append(k, v, slots, pos, *pools)
            ops.attend(q, start, lens, table, *pools, max(new), max_kv, out=out)

        step(w.ops)
        torch.cuda.synchronize()
        graph, ops = torch.cuda.CUDAGraph(), Kv4Ops(own, w.spec, side)
        with torch.cuda.graph(graph, stream=side):
            step(ops)
        for turn in range(2):
            big = World4(own, [2500], [64], D=128, P=64)
            big.attend(big.rows(big.Hq)[0].to(DEV), max_kv=200000 * (turn + 1))
            torch.cuda.synchronize()
            for x in (q, k, v):
                x.copy_(torch.randn(x.shape))
            step(w.ops)
            torch.cuda.synchronize()
            want = out.clone()
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
        own.sync_status()


def test_attention_on_several_streams_of_one_context():
    with Context(0) as own:
        worlds = [World4(own, [3000, 40, 700], [1, 1, 1], D=128, P=64), World4(own, [9000] * 8, [1] * 8, D=128, P=128, H=4, Hq=32),
                  World4(own, [2500], [64], D=64, P=16)]
        calls = []
        for w, (new, most) in zip(worlds, [(1, 3001), (1, 9001), (64, 20000)]):
            args = (w.rows(w.Hq)[0].to(DEV), *(w.dev(x, I32) for x in (w.start, w.kv_len, w.table)), *w.pools(), new, most)
            calls.append((w, args, w.ops.attend(*args).clone()))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in calls]
        for turn in range(4):
            got = []
            for _ in range(3):
                for i, (w, args, want) in enumerate(calls):
                    got.append((Kv4Ops(own, w.spec, streams[(i + turn) % 3]).attend(*args), want))
            torch.cuda.synchronize()
            assert all(torch.equal(x, want) for x, want in got)
        own.sync_status()


def test_server_loop():
    """Every request ends and gives its pages back. Half a step of a row of normal values is at most 7 / 30; it moves a score by
    sqrt(64) * 0.13 / 8 in root mean square, 0.65 at five times that, which moves weight of at most tanh(0.33) / 2 = 0.16 over
    a spread of at most 8: 1.3 + 0.24 in all."""
    from aihost_b200 import serve_kv8

    r = serve_kv8.main(["--batch", "5", "--requests", "9", "--layers", "2", "--prompt", "200", "--answer", "12", "--bits", "4"])
    assert r["free"] == r["pages"] and r["worst"] < 1.6


# ------------------------------------------------------------------------------------------------ refusals

def test_arguments_are_checked_in_python_too(ctx):
    w = World4(ctx, [20], [2])
    q, k = w.rows(w.Hq)[0].to(DEV), w.rows(w.H)[0].to(DEV)
    pools, slots = w.pools(), w.dev(w.slots)
    good = [k, k, slots, None, *pools]
    w.ops.append(*good)
    for i, bad in ((0, k.float()), (0, k[:1]), (1, k.cpu()), (2, slots.int()), (4, pools[0].char()), (4, pools[0][:, :, :, :-1]),
                   (6, pools[2].float()), (6, pools[2][..., 0]), (7, pools[3].cpu())):
        with pytest.raises(AttnError) as e:
            w.ops.append(*good[:i], bad, *good[i + 1:])
        assert e.value.status == A.EINVAL
    with pytest.raises(AttnError):
        w.ops.read(pools[0], pools[2], slots, torch.bfloat16)
    with pytest.raises(AttnError):
        w.ops.read(pools[0], pools[2][:-1], slots)
    args = [w.dev(x, I32) for x in (w.start, w.kv_len, w.table)]
    w.ops.attend(q, *args, *pools, 2, 22)
    for bad in (dict(out=q[:1]), dict(row_first=args[1]), dict(prefix_len=w.dev(w.kv_len)), dict(alibi_slopes=q[0, 0].float())):
        with pytest.raises(AttnError):
            w.ops.attend(q, *args, *pools, 2, 22, **bad)
    with pytest.raises(AttnError):
        w.ops.attend(q, *args, *pools, 0, 22)
    # rotated rows need positions
    rot = World4(ctx, [20], [2], mode=ROPE_NEOX)
    with pytest.raises(AttnError):
        rot.ops.append(k, k, slots, None, *rot.pools())
    ctx.sync_status()


def test_empty_calls(ctx):
    w = World4(ctx, [20], [2])
    none = torch.zeros(0, w.H, w.D, dtype=torch.float16, device=DEV)
    w.ops.append(none, none, torch.zeros(0, dtype=torch.int64, device=DEV), None, *w.pools())
    assert w.ops.read(*w.pools()[::2], torch.zeros(0, dtype=torch.int64, device=DEV)).shape == (0, w.H, w.D)
    ctx.sync_status()


def test_the_bounds_choose_the_kernel(ctx):
    """Between them the bounds of these tests run both kernels where both can."""
    w = World4(ctx, [20], [2], D=128)
    assert w.ops.plan(64, 64, 1, 8192)[1] == w.ops.plan(24, 100, 5, 9000)[1] == KV8_SPLIT_CACHE
    assert w.ops.plan(1, 2048, 2048, 16384)[1] == KV8_TENSOR
    for io in (F16, F32):
        for case in ("prompts", "prompts, d 128", "prompts, page 128", "prompt over old rows"):
            w = World4(ctx, io=io, **ATTENDS[case])
            kernels = {w.ops.plan(len(w.new), w.T, max(w.new), b or int(w.kv_len.max()))[1] for b in BOUNDS}
            assert (KV8_TENSOR in kernels) == (io == F16) and (io == F16 or KV8_SPLIT_CACHE in kernels)
