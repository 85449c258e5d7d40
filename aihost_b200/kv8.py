"""The 8-bit paged KV cache: int8 values with one scale per page and KV head.

It takes the place of the reference's unwired QuantizedKVCache (Inference/QuantizedKVCache.cs:46-133) and of
KVCache.Add's per-token Concat (InferenceEngine.cs:598-622), for batches of requests of uneven length:

  Kv8Ops.map_pages      one step's block tables, slots and positions, on the GPU   (aihost_page_map)
  Kv8Ops.release_pages  finished requests' pages back on the free stack            (aihost_page_release)
  Kv8Ops.append         the step's K (rotated) and V rows into the cache           (aihost_kv8_append)
  Kv8Ops.attend         attention of the step's query rows over the cache          (aihost_kv8_attention)
  Kv8Ops.read           cached rows as the values they stand for                   (aihost_kv8_read)
  Kv8Cache              pools, block table, lengths and free stack of a running batch, and its steps

Rows of a step lie one after another, sequence by sequence ("tokens"); lengths and tables stay on the device, and
the host gives upper bounds. Tensors are torch CUDA tensors on the context's device; their shapes, types and strides
are checked by the module _kv8 (built with the library), the rest by the library. Work is enqueued on `stream` (default: torch's current stream).
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import NamedTuple

import torch

from . import EINVAL, F16, F32, KV8_ROUND_Q, ROPE_INTERLEAVED, AttnError, Kv8Desc, check, lib
from .ops import Context

lib()  # the module below calls the same library
from . import _kv8  # noqa: E402

_kv8.set_error(AttnError)
_CODES = {torch.float32: F32, torch.float16: F16}


@dataclass
class Kv8Spec:
    """One layer over an 8-bit paged cache (aihost_kv8_desc; token strides are taken from the tensors)."""

    n_q_heads: int
    n_kv_heads: int
    head_dim: int
    page_rows: int = 64
    n_pages: int = 1
    max_pages: int = 1
    io_dtype: int = F16
    out_dtype: int = F16
    scale: float = 0.0
    score_cap: float = 0.0
    rope_theta: float = 10000.0
    rope_mode: int = ROPE_INTERLEAVED
    round_q: bool = False  # a rotated float16 q may be rounded to float16 (faster for prompts of head_dim 128)

    def desc(self) -> Kv8Desc:
        return Kv8Desc(self.n_q_heads, self.n_kv_heads, self.head_dim, self.page_rows, self.n_pages, self.max_pages,
                       self.io_dtype, self.out_dtype, self.scale, self.score_cap, self.rope_theta,
                       self.rope_mode | (KV8_ROUND_Q if self.round_q else 0), 0, 0)


class StepMap(NamedTuple):
    """What aihost_page_map gives for one step (device tensors)."""

    kv_len: torch.Tensor       # int32 [batch]: cached rows with this step's
    row_start: torch.Tensor    # int32 [batch + 1]: first token of every sequence
    slots: torch.Tensor        # int64 [max_tokens]: page * page_rows + row, -1 past the last token
    positions: torch.Tensor    # int32 [max_tokens]: row in the sequence
    free_count: torch.Tensor   # int32 [1]


class Kv8Ops:
    """The operators of one layer description on one context. `_kv8` checks the tensors and makes the calls."""

    def __init__(self, ctx: Context, spec: Kv8Spec, stream=None):
        self.ctx, self.spec, self.stream = ctx, spec, stream
        self.device = torch.device("cuda", ctx.device)
        self._desc = spec.desc()
        self._at = ctypes.addressof(self._desc)

    def _st(self) -> int | None:
        return None if self.stream is None else self.stream.cuda_stream

    def map_pages(self, seq_len: torch.Tensor, n_new: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
                  block_table: torch.Tensor, max_tokens: int, into: StepMap | None = None) -> StepMap:
        """One step's bookkeeping for seq_len, n_new (int32 [batch]): takes pages from the stack free_pages (its first
        free_count[0] entries are free), enters them in block_table (int32 [batch, max_pages], in place) and returns
        the step's StepMap; `into` names its tensors (kv_len may be seq_len, free_count may be free_count)."""
        return StepMap(*_kv8.map_pages(self.ctx.handle.value, self.ctx.device, self._at, self._st(), max_tokens, seq_len,
                                       n_new, free_pages, free_count, block_table, into))

    def release_pages(self, done: torch.Tensor, seq_len: torch.Tensor, free_pages: torch.Tensor,
                      free_count: torch.Tensor, block_table: torch.Tensor) -> None:
        """Ends the sequences with done != 0 (int32 [batch]): their pages go back on the stack, seq_len becomes 0."""
        _kv8.release_pages(self.ctx.handle.value, self.ctx.device, self._at, self._st(), done, seq_len, free_pages,
                           free_count, block_table)

    def append(self, k_new: torch.Tensor, v_new: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor | None,
               k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
        """Stores k_new (rotated at positions), v_new [n, n_kv_heads, head_dim] at slots (-1: skipped). Their tokens may
        lie apart, alike in both (columns of a fused projection's output)."""
        _kv8.append(self.ctx.handle.value, self.ctx.device, self._at, self._st(), k_new, v_new, slots, positions, k_pool,
                    v_pool, k_scale, v_scale)

    def read(self, pool: torch.Tensor, scale: torch.Tensor, slots: torch.Tensor, dtype: torch.dtype = torch.float16,
             out: torch.Tensor | None = None) -> torch.Tensor:
        """The rows at slots of one pool, [n, n_kv_heads, head_dim], as the values they stand for (zeros for -1)."""
        code = _CODES.get(dtype)
        if code is None:
            raise AttnError(EINVAL, f"unsupported dtype {dtype} (float32 or float16)")
        return _kv8.read(self.ctx.handle.value, self.ctx.device, self._at, self._st(), pool, scale, slots, code, out)

    def attend(self, q: torch.Tensor, row_start: torch.Tensor, kv_len: torch.Tensor, block_table: torch.Tensor,
               k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, max_new: int,
               max_kv: int, prefix_len: torch.Tensor | None = None, row_first: torch.Tensor | None = None,
               alibi_slopes: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of q [n, n_q_heads, head_dim] (rotated here) over the cache, [n, n_q_heads, head_dim]. max_new and
        max_kv: upper bounds on any sequence's new rows and on kv_len. prefix_len (int32 [batch]): cache rows that all
        rows of the sequence see; row_first (int32 [n]): the first cache row that a row sees; alibi_slopes (fp32
        [n_q_heads]): score - slope * distance. A row that sees nothing gets zeros; rows of no sequence (spare tokens, a
        refused step) are not computed, and hold what the memory held. The context's scratch grows on the
        first call that needs more (which waits for the GPU: make such a call before capturing a graph; graphs captured
        before keep the scratch they were captured with)."""
        return _kv8.attend(self.ctx.handle.value, self.ctx.device, self._at, self._st(), q, row_start, kv_len, block_table,
                           k_pool, v_pool, k_scale, v_scale, max_new, max_kv, prefix_len, row_first, alibi_slopes, out)

    def plan(self, batch: int, n_tokens: int, max_new: int, max_kv: int) -> tuple[int, int]:
        """(scratch bytes, KV8_SPLIT_CACHE or KV8_TENSOR) of an `attend` with these sizes and bounds."""
        need, kernel = ctypes.c_size_t(), ctypes.c_int32()
        check(lib().aihost_kv8_plan(self.ctx.handle, ctypes.byref(self._desc), batch, n_tokens, max_new, max_kv,
                                    ctypes.byref(need), ctypes.byref(kernel)))
        return need.value, kernel.value


class Kv8Cache:
    """Pools, block table, lengths and free pages of a running batch, with all bookkeeping on the GPU.

    A step: m = cache.begin(n_new, max_tokens); for every layer cache.append(layer, k, v) and
    cache.attend(layer, q, ...); cache.end(). `release` ends requests. Nothing here waits for the GPU: a step that runs out of
    pages is refused whole by the kernels (every slot -1, no rows) and reported by ctx.sync_status().

    With a `stream`, the cache's tensors are made on it and all its work runs on it; what the caller hands in (n_new, q, k,
    v) has to be ready on that stream and to stay alive until its work is done, as with any stream of torch's."""

    def __init__(self, ctx: Context, spec: Kv8Spec, batch: int, n_layers: int = 1, stream=None):
        self.ctx, self.spec, self.batch = ctx, spec, batch
        self.ops = self._make_ops(ctx, spec, stream)
        dev = self.ops.device
        with torch.cuda.stream(stream):  # filled, and given back, in the order of the steps' work
            self._make_pools(n_layers, dev)
            self.block_table = torch.full((batch, spec.max_pages), -1, dtype=torch.int32, device=dev)
            self.free_pages = torch.arange(spec.n_pages - 1, -1, -1, dtype=torch.int32, device=dev)
            self.free_count = torch.full((1,), spec.n_pages, dtype=torch.int32, device=dev)
            self.seq_len = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.map: StepMap | None = None

    _make_ops = Kv8Ops

    def _make_pools(self, n_layers: int, dev: torch.device) -> None:
        spec = self.spec
        pool = (spec.n_pages, spec.n_kv_heads, spec.page_rows, spec.head_dim)
        self.k = [torch.zeros(pool, dtype=torch.int8, device=dev) for _ in range(n_layers)]
        self.v = [torch.zeros(pool, dtype=torch.int8, device=dev) for _ in range(n_layers)]
        self.k_scale = [torch.zeros(pool[:2], device=dev) for _ in range(n_layers)]
        self.v_scale = [torch.zeros(pool[:2], device=dev) for _ in range(n_layers)]

    def _layer(self, layer: int) -> tuple[torch.Tensor, ...]:
        return self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer]

    def begin(self, n_new: torch.Tensor, max_tokens: int) -> StepMap:
        """Pages, slots and positions for n_new (int32 [batch]) more rows of every sequence."""
        if self.map is not None:
            raise AttnError(EINVAL, "the step before has not ended")
        self.map = self.ops.map_pages(self.seq_len, n_new, self.free_pages, self.free_count, self.block_table, max_tokens)
        self.free_count = self.map.free_count
        return self.map

    def _step(self) -> StepMap:
        if self.map is None:
            raise AttnError(EINVAL, "no step has begun")
        return self.map

    def append(self, layer: int, k_new: torch.Tensor, v_new: torch.Tensor) -> None:
        m = self._step()
        self.ops.append(k_new, v_new, m.slots, m.positions, *self._layer(layer))

    def attend(self, layer: int, q: torch.Tensor, max_new: int, max_kv: int, **kw) -> torch.Tensor:
        m = self._step()
        return self.ops.attend(q, m.row_start, m.kv_len, self.block_table, *self._layer(layer), max_new, max_kv, **kw)

    def end(self) -> None:
        """Commits the step's rows (after its last layer)."""
        self.seq_len = self._step().kv_len
        self.map = None

    def release(self, done: torch.Tensor) -> None:
        """Ends the sequences with done != 0 (int32 [batch]), between steps."""
        if self.map is not None:
            raise AttnError(EINVAL, "the step before has not ended")
        self.ops.release_pages(done, self.seq_len, self.free_pages, self.free_count, self.block_table)


__all__ = ["Kv8Spec", "Kv8Ops", "Kv8Cache", "StepMap"]
