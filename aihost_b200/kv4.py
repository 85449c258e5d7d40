"""The 4-bit paged KV cache: codes of 4 bits with an fp16 pair (low, step) for each row of a KV head.

Pages, steps, masks and calls are those of the 8-bit cache (kv8.py), with half the bytes:

  Kv4Ops.map_pages, release_pages   as Kv8Ops has them
  Kv4Ops.append    the step's K (rotated) and V rows into the cache           (aihost_kv4_append)
  Kv4Ops.attend    attention of the step's query rows over the cache          (aihost_kv4_attention)
  Kv4Ops.read      cached rows as the values they stand for                   (aihost_kv4_read)
  Kv4Cache         pools, block table, lengths and free stack of a running batch, and its steps

A code c of a row stands for low + step * c, as in GGUF's Q4_1 with a row in place of its 32 values. A row is
stored by itself: an append changes no other row, and its tokens need no order. Layouts: pools uint8
[n_pages, n_kv_heads, page_rows, head_dim / 2] (the order of the nibbles is in include/aihost_attn.h), ranges float16
[n_pages, n_kv_heads, page_rows, 2].
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import EINVAL, AttnError, check, lib
from .kv8 import _CODES, Kv8Cache, Kv8Ops, Kv8Spec, StepMap, _kv8


@dataclass
class Kv4Spec(Kv8Spec):
    """One layer over a 4-bit paged cache: the fields of Kv8Spec."""


class Kv4Ops(Kv8Ops):
    """The operators of one layer description on one context."""

    def append(self, k_new: torch.Tensor, v_new: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor | None,
               k_pool: torch.Tensor, v_pool: torch.Tensor, k_range: torch.Tensor, v_range: torch.Tensor) -> None:
        """Stores k_new (rotated at positions), v_new [n, n_kv_heads, head_dim] at slots (-1: skipped; each other slot
        once). Their tokens may lie apart, alike in both (columns of a fused projection's output)."""
        _kv8.append4(self.ctx.handle.value, self.ctx.device, self._at, self._st(), k_new, v_new, slots, positions, k_pool,
                     v_pool, k_range, v_range)

    def read(self, pool: torch.Tensor, range: torch.Tensor, slots: torch.Tensor, dtype: torch.dtype = torch.float16,
             out: torch.Tensor | None = None) -> torch.Tensor:
        """The rows at slots of one pool, [n, n_kv_heads, head_dim], as the values they stand for (zeros for -1)."""
        code = _CODES.get(dtype)
        if code is None:
            raise AttnError(EINVAL, f"unsupported dtype {dtype} (float32 or float16)")
        return _kv8.read4(self.ctx.handle.value, self.ctx.device, self._at, self._st(), pool, range, slots, code, out)

    def attend(self, q: torch.Tensor, row_start: torch.Tensor, kv_len: torch.Tensor, block_table: torch.Tensor,
               k_pool: torch.Tensor, v_pool: torch.Tensor, k_range: torch.Tensor, v_range: torch.Tensor, max_new: int,
               max_kv: int, prefix_len: torch.Tensor | None = None, row_first: torch.Tensor | None = None,
               alibi_slopes: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of q [n, n_q_heads, head_dim] (rotated here) over the cache, [n, n_q_heads, head_dim]; arguments,
        masks, rows left as they are and the context's scratch as for Kv8Ops.attend."""
        return _kv8.attend4(self.ctx.handle.value, self.ctx.device, self._at, self._st(), q, row_start, kv_len, block_table,
                            k_pool, v_pool, k_range, v_range, max_new, max_kv, prefix_len, row_first, alibi_slopes, out)

    def plan(self, batch: int, n_tokens: int, max_new: int, max_kv: int) -> tuple[int, int]:
        """(scratch bytes, KV8_SPLIT_CACHE or KV8_TENSOR) of an `attend` with these sizes and bounds."""
        need, kernel = ctypes.c_size_t(), ctypes.c_int32()
        check(lib().aihost_kv4_plan(self.ctx.handle, ctypes.byref(self._desc), batch, n_tokens, max_new, max_kv,
                                    ctypes.byref(need), ctypes.byref(kernel)))
        return need.value, kernel.value


class Kv4Cache(Kv8Cache):
    """Kv8Cache over 4-bit pools: begin, append, attend, end and release as there."""

    _make_ops = Kv4Ops

    def _make_pools(self, n_layers: int, dev: torch.device) -> None:
        spec = self.spec
        pool = (spec.n_pages, spec.n_kv_heads, spec.page_rows)
        self.k = [torch.zeros(*pool, spec.head_dim // 2, dtype=torch.uint8, device=dev) for _ in range(n_layers)]
        self.v = [torch.zeros(*pool, spec.head_dim // 2, dtype=torch.uint8, device=dev) for _ in range(n_layers)]
        self.k_range = [torch.zeros(*pool, 2, dtype=torch.float16, device=dev) for _ in range(n_layers)]
        self.v_range = [torch.zeros(*pool, 2, dtype=torch.float16, device=dev) for _ in range(n_layers)]

    def _layer(self, layer: int) -> tuple[torch.Tensor, ...]:
        return self.k[layer], self.v[layer], self.k_range[layer], self.v_range[layer]


__all__ = ["Kv4Spec", "Kv4Ops", "Kv4Cache", "StepMap"]
