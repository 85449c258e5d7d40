"""Which kernel the 4-bit cache's attention runs, what it keeps of a rotated q, and whether the calls that other tests only repeat are
right. Bounds as in test_gpu_kv4.py."""
import dataclasses

import numpy as np
import pytest

from aihost_b200 import KV8_SPLIT_CACHE, KV8_TENSOR, ROPE_INTERLEAVED, ROPE_NEOX, ROPE_NONE
from aihost_b200.kv4 import Kv4Ops
from test_gpu_kv4 import World4
from test_gpu_kv8 import ATTENDS, BOUNDS, DEV

pytestmark = pytest.mark.gpu


def _kernel(w, max_kv):
    return w.ops.plan(len(w.new), w.T, max(w.new), max_kv or int(w.kv_len.max()))[1]


@pytest.mark.parametrize("case", ["prompts", "prompts, d 128", "prompts, page 128", "prompt over old rows"])
def test_the_bounds_run_both_kernels(ctx, case):
    """Prompts of fp16 tensors: what the two bounds of the attention tests are for."""
    w = World4(ctx, **ATTENDS[case])
    assert {_kernel(w, b) for b in BOUNDS} == {KV8_SPLIT_CACHE, KV8_TENSOR}


@pytest.mark.parametrize("rounded", [False, True])
@pytest.mark.parametrize("max_kv", [None, 40000])
@pytest.mark.parametrize("what", ["plain", "cap", "bias", "documents", "one row"])
@pytest.mark.parametrize("D, mode", [(64, ROPE_NEOX), (128, ROPE_INTERLEAVED), (128, ROPE_NEOX)])
def test_rotated_prompts_of_either_precision(ctx, D, mode, what, max_kv, rounded):
    """round_q: the tcgen05 kernel with head_dim 128 rounds a rotated q to fp16, whose error 2^-11 a score then has of sum |q| kmax; no
    other call does."""
    cached, new = ([700, 5], [1, 300]) if what == "one row" else ([700, 0, 40], [300, 129, 17])
    w = World4(ctx, cached, new, Hq=8, H=1, D=D, P=32, mode=mode, cap=6.0 if what == "cap" else 0.0, seed=62)
    w.spec = dataclasses.replace(w.spec, round_q=rounded)
    w.ops = Kv4Ops(ctx, w.spec)
    first = slopes = None
    if what == "bias":
        slopes = [2.0 ** -(h + 1) for h in range(8)]
    if what == "documents":  # rows 0..15 of a sequence look back to its start, the later ones to their own neighbours
        first = [0 if i < 16 else max(0, int(p) - 20) for n, c in zip(new, cached) for i, p in enumerate(range(c, c + n))]
    assert max_kv is None or _kernel(w, max_kv) == KV8_TENSOR
    q, q64 = w.rows(w.Hq)
    out = w.attend(q.to(DEV), max_kv=max_kv, first=first, slopes=slopes).double().cpu().numpy()
    ctx.sync_status()
    ref, off, most, size = w.reference(q64, first=first, slopes=slopes)
    lost = rounded and D == 128 and _kernel(w, max_kv) == KV8_TENSOR
    ds = size[..., None] * (2.0 ** -18 + (2.0 ** -11 if lost else 0.0))
    tol = 2.0 ** -11 * np.abs(ref) + off * 2.0 ** -11 + most * (2.0 ** -16 + 2 * ds) + 1e-7
    assert (np.abs(out - ref) <= tol).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mode", [ROPE_NONE, ROPE_NEOX])
@pytest.mark.parametrize("shape", [dict(cached=[700, 1], new=[64, 255], Hq=8), dict(cached=[127, 1], new=[130, 255], Hq=6)])
def test_the_calls_repeated_from_cold_caches_are_right(ctx, D, mode, shape):
    World4(ctx, H=2, D=D, P=128, mode=mode, seed=17, **shape).check(ctx, max_kv=100000)


def test_server_loop_against_the_cached_rows():
    """Values of about N(0, 1), at most 5 in size, steps of at most 0.36: 2^-11 of a result, 2^-11 of 7.5 steps for the weights, and for
    the scores' error, 2^-18 of sum |q| kmax = 64 * 0.8 * 3.5 / 8, twice that of 5: 4.6e-3 in all."""
    from aihost_b200 import serve_kv8

    r = serve_kv8.main(["--batch", "5", "--requests", "9", "--layers", "2", "--prompt", "200", "--answer", "12", "--bits", "4"])
    assert r["free"] == r["pages"] and r["off_cached"] < 5e-3
