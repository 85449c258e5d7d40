"""Prompts over the 8-bit cache when neither instructions nor data are in any cache: every call gives the same bits."""
import pytest
import torch

from aihost_b200 import KV8_TENSOR, ROPE_NEOX, ROPE_NONE
from test_gpu_kv8 import DEV, I32, World

pytestmark = pytest.mark.gpu


def cold_calls(w, factors, n):
    """How many of n calls on fresh copies of the inputs, each after the caches were overwritten, differ from the first."""
    q = w.rows(w.Hq)[0].to(DEV)
    args = [q, *(w.dev(x, I32) for x in (w.start, w.kv_len, w.table)), *(w.dev(x) for x in factors)]
    assert w.ops.plan(len(w.new), w.T, max(w.new), 100000)[1] == KV8_TENSOR
    first, flush, other = w.ops.attend(*args, max(w.new), 100000), torch.empty(200 << 20, dtype=torch.uint8, device=DEV), 0
    for i in range(n):
        flush.fill_(i & 255)
        other += not torch.equal(w.ops.attend(*[x.clone() for x in args], max(w.new), 100000), first)
    return other


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mode", [ROPE_NONE, ROPE_NEOX])
def test_calls_from_cold_caches(ctx, D, mode):
    w = World(ctx, [700, 1], [64, 255], Hq=8, H=2, D=D, P=128, mode=mode, seed=17)
    assert cold_calls(w, (w.k, w.v, w.ks, w.vs), 1000) == 0
    ctx.sync_status()
