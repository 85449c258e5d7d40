"""Kernels that read a TMA ring in shared memory by plain loads and give a place back for the next copy, called when neither
instructions nor data are in any cache: every call gives the same bits, those of the first are checked."""
import pytest
import torch

from aihost_b200 import F16, Q4_K, Q5_K, Q8_0, ROPE_NEOX, gen
from aihost_b200.configs import CONFIGS, make_inputs
from aihost_b200.ops import ComputeOps, KVCache, WeightOps
from helpers import max_abs, oracle_forward
from test_gpu_weights import exact_bound_check

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
CALLS = 200


def _differing(call, flush):
    """(the first call's result, how many of CALLS more differ from it), each after the caches were overwritten."""
    first, other = call().clone(), 0
    for i in range(CALLS):
        flush.fill_(i & 255)
        other += not torch.equal(call(), first)
    return first, other


# 9000 and 3000 rows: every block goes round its ring. Groups of up to 8 query heads, of more, and more KV heads than the
# schedule over all sequences' tiles takes
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kv, hq, hkv, lengths", [
    (Q8_0, 16, 2, [9000, 3000]), (Q8_0, 16, 1, [9000, 3000]), (Q8_0, 72, 72, [3000]),
    (F16, 16, 2, [9000, 3000]), (F16, 16, 1, [9000, 3000])])
def test_decode_from_cold_caches(ctx, kv, hq, hkv, lengths, d):
    cfg = CONFIGS[5 if kv == Q8_0 else 3].scaled(batch=len(lengths), n_q_heads=hq, n_kv_heads=hkv, head_dim=d,
                                                 rope_mode=ROPE_NEOX, cached=None, cached_range=None, cached_list=lengths)
    inp, ops = make_inputs(cfg), ComputeOps(ctx)
    q, k_new, v_new = (inp[n].to(DEV) for n in ("q", "k_new", "v_new"))
    cache = KVCache(ctx, cfg.spec(inp["capacity"]), batch=cfg.batch, device=DEV)
    cache.k[0], cache.v[0], cache.seq_len = (inp[n].to(DEV).clone() for n in ("k_cache", "v_cache", "seq_len"))
    cache.host_len = list(inp["lengths"])

    def call():  # the append of every call writes the same row to the same place
        return ops.attention_layer(q, k_new, v_new, cache)

    first, other = _differing(call, torch.empty(200 << 20, dtype=torch.uint8, device=DEV))
    ctx.sync_status()
    ref = oracle_forward(cfg, inp)[0]
    assert other == 0 and max_abs(first.float().cpu().numpy(), ref) <= 2e-3


@pytest.mark.parametrize("kind", [Q4_K, Q5_K])
def test_weight_products_from_cold_caches(ctx, kind):
    """k split over at most eight blocks: the two-place ring of super-blocks goes round four times in each."""
    rows, k, n_out = 64, 16384, 1024
    a, ops = gen.normal((rows, k), 5, "a", dtype=torch.float16), WeightOps(ctx)
    w, a_dev = gen.kquant_blocks(kind, n_out * k // 256, 5, "w").to(DEV), a.to(DEV)

    def call():
        return ops.mat_mul_weights(a_dev, w, kind, n_out, out_dtype=torch.float32)

    first, other = _differing(call, torch.empty(200 << 20, dtype=torch.uint8, device=DEV))
    ctx.sync_status()
    w16 = ops.dequantize(w, kind, n_out * k, torch.float16).cpu().numpy().reshape(n_out, k)
    exact_bound_check(first.cpu().numpy(), a.numpy(), w16, False)
    assert other == 0
