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
are checked here, the rest by the library. Work is enqueued on `stream` (default: torch's current stream).
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import EINVAL, F16, F32, ROPE_INTERLEAVED, AttnError, Kv8Desc, check, lib
from .ops import Context

_TORCH = {F32: torch.float32, F16: torch.float16}


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

    def desc(self) -> Kv8Desc:
        return Kv8Desc(self.n_q_heads, self.n_kv_heads, self.head_dim, self.page_rows, self.n_pages, self.max_pages,
                       self.io_dtype, self.out_dtype, self.scale, self.score_cap, self.rope_theta, self.rope_mode, 0, 0)


@dataclass
class StepMap:
    """What aihost_page_map gives for one step (device tensors)."""

    kv_len: torch.Tensor       # int32 [batch]: cached rows with this step's
    row_start: torch.Tensor    # int32 [batch + 1]: first token of every sequence
    slots: torch.Tensor        # int64 [max_tokens]: page * page_rows + row, -1 past the last token
    positions: torch.Tensor    # int32 [max_tokens]: row in the sequence
    free_count: torch.Tensor   # int32 [1]


class Kv8Ops:
    """The operators of one layer description on one context."""

    def __init__(self, ctx: Context, spec: Kv8Spec, stream=None):
        self.ctx, self.spec, self.stream = ctx, spec, stream
        self.device = torch.device("cuda", ctx.device)
        self._desc = spec.desc()
        self._ref = ctypes.byref(self._desc)
        self._lib = lib()
        self._pool = (spec.n_pages, spec.n_kv_heads, spec.page_rows, spec.head_dim)
        self._need: dict = {}  # scratch bytes by the sizes of a call

    # ---- argument checks

    def _st(self):
        return (self.stream or torch.cuda.current_stream(self.device)).cuda_stream

    def _array(self, t: torch.Tensor | None, name: str, dtype: torch.dtype, shape: tuple | None = None,
               at_least: int | None = None) -> int | None:
        if t is None:
            return None
        if t.dtype != dtype or t.device != self.device or not t.is_contiguous():
            raise AttnError(EINVAL, f"{name} must be a contiguous {dtype} tensor on {self.device}")
        if shape is not None and t.shape != shape:
            raise AttnError(EINVAL, f"{name} must have shape {shape}, not {tuple(t.shape)}")
        if at_least is not None and t.numel() < at_least:
            raise AttnError(EINVAL, f"{name} must have at least {at_least} elements, not {t.numel()}")
        return t.data_ptr()

    def _rows(self, t: torch.Tensor, name: str, heads: int) -> int:
        """Bytes between tokens of t [n, heads, head_dim], whose rows may lie apart (a fused projection's output)."""
        d = self.spec.head_dim
        if t.dtype != _TORCH[self.spec.io_dtype] or t.device != self.device or t.dim() != 3 or t.shape[1:] != (heads, d):
            raise AttnError(EINVAL, f"{name} must be {_TORCH[self.spec.io_dtype]} [n, {heads}, {d}] on {self.device}")
        packed = heads * d
        if t.shape[0] == 0:
            return packed * t.element_size()
        if t.stride(2) != 1 or (heads > 1 and t.stride(1) != d) or (t.shape[0] > 1 and t.stride(0) < packed):
            raise AttnError(EINVAL, f"{name} must have its heads packed within a token, and tokens in order")
        return (t.stride(0) if t.shape[0] > 1 else packed) * t.element_size()

    # ---- operators

    def map_pages(self, seq_len: torch.Tensor, n_new: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
                  block_table: torch.Tensor, max_tokens: int, into: StepMap | None = None) -> StepMap:
        """One step's bookkeeping for seq_len, n_new (int32 [batch]): takes pages from the stack free_pages (its first
        free_count[0] entries are free), enters them in block_table (int32 [batch, max_pages], in place) and returns
        the step's StepMap; `into` names its tensors (kv_len may be seq_len, free_count may be free_count)."""
        s, n = self.spec, seq_len.numel()
        if into is None:
            new = lambda k, dt=torch.int32: torch.empty(k, dtype=dt, device=self.device)  # noqa: E731
            into = StepMap(new(n), new(n + 1), new(max_tokens, torch.int64), new(max_tokens), new(1))
        i32 = torch.int32
        check(self._lib.aihost_page_map(
            self.ctx.handle, n, s.page_rows, s.n_pages, s.max_pages, max_tokens,
            self._array(seq_len, "seq_len", i32, (n,)), self._array(n_new, "n_new", i32, (n,)),
            self._array(free_pages, "free_pages", i32, at_least=s.n_pages),
            self._array(free_count, "free_count", i32, (1,)),
            self._array(block_table, "block_table", i32, (n, s.max_pages)), self._array(into.kv_len, "kv_len", i32, (n,)),
            self._array(into.row_start, "row_start", i32, (n + 1,)),
            self._array(into.slots, "slots", torch.int64, at_least=max_tokens),
            self._array(into.positions, "positions", i32, at_least=max_tokens),
            self._array(into.free_count, "free_count", i32, (1,)), self._st()))
        return into

    def release_pages(self, done: torch.Tensor, seq_len: torch.Tensor, free_pages: torch.Tensor,
                      free_count: torch.Tensor, block_table: torch.Tensor) -> None:
        """Ends the sequences with done != 0 (int32 [batch]): their pages go back on the stack, seq_len becomes 0."""
        s, n, i32 = self.spec, seq_len.numel(), torch.int32
        check(self._lib.aihost_page_release(
            self.ctx.handle, n, s.page_rows, s.n_pages, s.max_pages, self._array(done, "done", i32, (n,)),
            self._array(seq_len, "seq_len", i32, (n,)), self._array(block_table, "block_table", i32, (n, s.max_pages)),
            self._array(free_pages, "free_pages", i32, at_least=s.n_pages),
            self._array(free_count, "free_count", i32, (1,)), self._st()))

    def append(self, k_new: torch.Tensor, v_new: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor | None,
               k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
        """Stores k_new (rotated at positions), v_new [n, n_kv_heads, head_dim] at slots (-1: skipped)."""
        s, n = self.spec, k_new.shape[0]
        stride = self._rows(k_new, "k_new", s.n_kv_heads)
        if v_new.shape[0] != n or self._rows(v_new, "v_new", s.n_kv_heads) != stride:
            raise AttnError(EINVAL, "k_new and v_new must have the same tokens and the same stride between them")
        self._desc.kv_token_stride = stride
        per_page, i8, f32 = self._pool[:2], torch.int8, torch.float32
        check(self._lib.aihost_kv8_append(
            self.ctx.handle, self._ref, n, k_new.data_ptr(), v_new.data_ptr(),
            self._array(slots, "slots", torch.int64, at_least=n), self._array(positions, "positions", torch.int32, at_least=n),
            self._array(k_pool, "k_pool", i8, self._pool), self._array(v_pool, "v_pool", i8, self._pool),
            self._array(k_scale, "k_scale", f32, per_page), self._array(v_scale, "v_scale", f32, per_page), self._st()))

    def read(self, pool: torch.Tensor, scale: torch.Tensor, slots: torch.Tensor, dtype: torch.dtype = torch.float16,
             out: torch.Tensor | None = None) -> torch.Tensor:
        """The rows at slots of one pool, [n, n_kv_heads, head_dim], as the values they stand for (zeros for -1)."""
        s, n = self.spec, slots.numel()
        if dtype not in (torch.float16, torch.float32):
            raise AttnError(EINVAL, f"unsupported dtype {dtype} (float32 or float16)")
        shape = (n, s.n_kv_heads, s.head_dim)
        if out is None:
            out = torch.empty(shape, dtype=dtype, device=self.device)
        check(self._lib.aihost_kv8_read(
            self.ctx.handle, self._ref, n, self._array(slots, "slots", torch.int64),
            self._array(pool, "pool", torch.int8, self._pool),
            self._array(scale, "scale", torch.float32, self._pool[:2]), self._array(out, "out", dtype, shape),
            F16 if dtype == torch.float16 else F32, self._st()))
        return out

    def attend(self, q: torch.Tensor, row_start: torch.Tensor, kv_len: torch.Tensor, block_table: torch.Tensor,
               k_pool: torch.Tensor, v_pool: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, max_new: int,
               max_kv: int, prefix_len: torch.Tensor | None = None, row_first: torch.Tensor | None = None,
               alibi_slopes: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of q [n, n_q_heads, head_dim] (rotated here) over the cache, [n, n_q_heads, head_dim]. max_new and
        max_kv: upper bounds on any sequence's new rows and on kv_len. prefix_len (int32 [batch]): cache rows that all
        rows of the sequence see; row_first (int32 [n]): the first cache row that a row sees; alibi_slopes (fp32
        [n_q_heads]): score - slope * distance. A row that sees nothing gets zeros."""
        s, n, b = self.spec, q.shape[0], kv_len.numel()
        self._desc.q_token_stride = self._rows(q, "q", s.n_q_heads)
        odt = _TORCH[s.out_dtype]
        if out is None:
            out = torch.empty(n, s.n_q_heads, s.head_dim, dtype=odt, device=self.device)
        key = (b, n, max_new, max_kv)
        need = self._need.get(key)
        if need is None:
            size = ctypes.c_size_t()
            check(self._lib.aihost_kv8_workspace_size(self._ref, b, n, max_new, max_kv, ctypes.byref(size)))
            if len(self._need) >= 4096:
                self._need.clear()
            need = self._need[key] = size.value
        if need > self.ctx.reserved:
            self.ctx.reserve(need)
        per_page, i8, i32, f32 = self._pool[:2], torch.int8, torch.int32, torch.float32
        check(self._lib.aihost_kv8_attention(
            self.ctx.handle, self._ref, b, n, max_new, max_kv, q.data_ptr(), self._array(row_start, "row_start", i32, (b + 1,)),
            self._array(kv_len, "kv_len", i32, (b,)), self._array(block_table, "block_table", i32, (b, s.max_pages)),
            self._array(k_pool, "k_pool", i8, self._pool), self._array(v_pool, "v_pool", i8, self._pool),
            self._array(k_scale, "k_scale", f32, per_page), self._array(v_scale, "v_scale", f32, per_page),
            self._array(prefix_len, "prefix_len", i32, (b,)), self._array(row_first, "row_first", i32, at_least=n),
            self._array(alibi_slopes, "alibi_slopes", f32, (s.n_q_heads,)),
            self._array(out, "out", odt, (n, s.n_q_heads, s.head_dim)), self._st()))
        return out


class Kv8Cache:
    """Pools, block table, lengths and free pages of a running batch, with all bookkeeping on the GPU.

    A step: m = cache.begin(n_new, max_tokens); for every layer cache.append(layer, k, v) and
    cache.attend(layer, q, ...); cache.end(). `release` ends requests. Nothing here waits for the GPU: a step that runs out of
    pages is refused whole by the kernels (every slot -1, no rows) and reported by ctx.sync_status()."""

    def __init__(self, ctx: Context, spec: Kv8Spec, batch: int, n_layers: int = 1, stream=None):
        self.ctx, self.spec, self.batch = ctx, spec, batch
        self.ops = Kv8Ops(ctx, spec, stream)
        dev, pool = self.ops.device, (spec.n_pages, spec.n_kv_heads, spec.page_rows, spec.head_dim)
        self.k = [torch.zeros(pool, dtype=torch.int8, device=dev) for _ in range(n_layers)]
        self.v = [torch.zeros(pool, dtype=torch.int8, device=dev) for _ in range(n_layers)]
        self.k_scale = [torch.zeros(pool[:2], device=dev) for _ in range(n_layers)]
        self.v_scale = [torch.zeros(pool[:2], device=dev) for _ in range(n_layers)]
        self.block_table = torch.full((batch, spec.max_pages), -1, dtype=torch.int32, device=dev)
        self.free_pages = torch.arange(spec.n_pages - 1, -1, -1, dtype=torch.int32, device=dev)
        self.free_count = torch.full((1,), spec.n_pages, dtype=torch.int32, device=dev)
        self.seq_len = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.map: StepMap | None = None

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
        self.ops.append(k_new, v_new, m.slots, m.positions, self.k[layer], self.v[layer], self.k_scale[layer],
                        self.v_scale[layer])

    def attend(self, layer: int, q: torch.Tensor, max_new: int, max_kv: int, **kw) -> torch.Tensor:
        m = self._step()
        return self.ops.attend(q, m.row_start, m.kv_len, self.block_table, self.k[layer], self.v[layer],
                               self.k_scale[layer], self.v_scale[layer], max_new, max_kv, **kw)

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
