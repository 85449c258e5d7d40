"""A small server loop over the 8-bit or the 4-bit paged cache: python -m aihost_b200.serve_kv8 [--bits 4]

Requests of uneven prompt and answer lengths come and go in a fixed batch. Every step feeds the rows of all running
requests (whole prompts beside single tokens) through a stack of attention layers with random weights: the weight
products (aihost_matmul_weights), the append and the attention; pages are assigned and freed on the GPU. One layer's
attention is checked at the end against attention over the same rows in fp32, unquantised, and with 4 bits, whose rows never
change, also against that over the rows that the cache holds."""
from __future__ import annotations

import argparse
import random
import time

import torch

from . import F16
from .kv4 import Kv4Cache, Kv4Spec
from .kv8 import Kv8Cache, Kv8Spec
from .ops import Context, WeightOps


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--requests", type=int, default=48)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=600, help="longest prompt")
    ap.add_argument("--answer", type=int, default=64, help="longest answer")
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--bits", type=int, choices=(4, 8), default=8, help="of the cache's values")
    a = ap.parse_args(argv)
    Hq, H, D, P = 14, 2, 64, 64  # a small model's heads
    width, dev = Hq * D, torch.device("cuda", 0)
    rng, g = random.Random(a.seed), torch.Generator(device=dev).manual_seed(a.seed)
    pages = -(-(a.prompt + a.answer) // P)
    with Context(0) as ctx:
        make_spec, make_cache = (Kv4Spec, Kv4Cache) if a.bits == 4 else (Kv8Spec, Kv8Cache)
        spec = make_spec(Hq, H, D, P, n_pages=a.batch * pages, max_pages=pages, rope_theta=1e6)
        cache, weights = make_cache(ctx, spec, a.batch, a.layers), WeightOps(ctx)
        w = lambda n, k: (torch.randn(n, k, generator=g, device=dev) / k ** 0.5).half()  # noqa: E731
        w_qkv = [w((Hq + 2 * H) * D, width) for _ in range(a.layers)]
        w_out = [w(width, width) for _ in range(a.layers)]
        left = a.requests
        todo = [0] * a.batch    # rows still to come for each place in the batch (its prompt counts as one step)
        lens = [0] * a.batch
        kept = [[] for _ in range(a.batch)]  # layer 0's K and V rows of place 0, for the check
        tokens = steps = 0
        worst, off_cached, began = 0.0, 0.0, time.perf_counter()
        while True:
            new = []
            for b in range(a.batch):
                if todo[b] == 0 and left:
                    left -= 1
                    todo[b] = rng.randint(1, a.answer)
                    kept[b] = []
                    new.append(rng.randint(1, a.prompt))
                else:
                    new.append(1 if todo[b] else 0)
            T = sum(new)
            if T == 0:
                break
            x = torch.randn(T, width, generator=g, device=dev).half()
            m = cache.begin(torch.tensor(new, dtype=torch.int32, device=dev), T)
            for layer in range(a.layers):
                qkv = weights.mat_mul_weights(x, w_qkv[layer], F16, (Hq + 2 * H) * D).view(T, Hq + 2 * H, D)
                q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
                cache.append(layer, k, v)
                o = cache.attend(layer, q, max(new), max(c + n for c, n in zip(lens, new)))
                if layer == 0 and new[0]:
                    pools = zip((cache.k, cache.v), (cache.k_range, cache.v_range)) if a.bits == 4 else ()
                    held = [cache.ops.read(p[0], r[0], m.slots[:new[0]], torch.float32) for p, r in pools]
                    kept[0].append((q[:new[0]], o[:new[0]], k[:new[0]], v[:new[0]], *held))
                x = x + weights.mat_mul_weights(o.view(T, width), w_out[layer], F16, width)
            cache.end()
            done = []
            for b in range(a.batch):
                lens[b] += new[b]
                todo[b] -= 1 if new[b] else 0
                done.append(1 if new[b] and todo[b] == 0 else 0)
                lens[b] = 0 if done[b] else lens[b]
            if done[0]:
                off = _check(ctx, kept[0], spec)
                worst, off_cached = max(worst, off[0]), max(off_cached, off[-1])
            cache.release(torch.tensor(done, dtype=torch.int32, device=dev))
            tokens, steps = tokens + T, steps + 1
        ctx.sync_status()
        took = time.perf_counter() - began
        free = cache.free_count.item()
    print(f"{a.requests} requests, {tokens} tokens in {steps} steps of {a.layers} layers: {took:.2f} s; "
          f"free pages at the end {free} of {spec.n_pages}; attention off the unquantised fp32 one by {worst:.4f} at most" +
          (f", off that over the cached rows by {off_cached:.4f}" if a.bits == 4 else ""))
    return {"tokens": tokens, "steps": steps, "free": free, "pages": spec.n_pages, "worst": worst,
            **({"off_cached": off_cached} if a.bits == 4 else {})}


def _check(ctx: Context, kept: list, spec: Kv8Spec) -> list[float]:
    """Largest difference of one request's attention outputs from attention in fp32 over its own rows, and over the rows as
    the cache holds them (rotated) where `kept` has those."""
    from .ops import ComputeOps

    q, o, *rows = (torch.cat(x).float().contiguous() for x in zip(*kept))
    n = q.shape[0]
    ops = ComputeOps(ctx)
    for x, heads in ((q, spec.n_q_heads), (rows[0], spec.n_kv_heads)):
        ops.apply_rope_full(x.view(n, -1), 0, heads, spec.head_dim, spec.rope_theta)
    off = []
    for k, v in zip(rows[0::2], rows[1::2]):
        k, v = (x.repeat_interleave(spec.n_q_heads // spec.n_kv_heads, 1) for x in (k, v))
        s = torch.einsum("thd,jhd->htj", q, k) / spec.head_dim ** 0.5
        s = s.masked_fill(torch.ones(n, n, device=q.device).triu(1).bool(), -torch.inf).softmax(-1)
        off.append((torch.einsum("htj,jhd->thd", s, v) - o).abs().max().item())
    return off


if __name__ == "__main__":
    main()
