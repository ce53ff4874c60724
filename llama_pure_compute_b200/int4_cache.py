"""4-bit KV caches with the step interface of ``KVCacheManager`` and
``RaggedKVCache``: ``LlamaForCausalLM`` and the generators take either.

The reference's ``Precision.INT4`` (src/llama_pure_compute/config.py:27-60) only
sizes a cache; here its rows are held in 4 bits (``ops.Int4KV``: 72 bytes a row
of 128 dims against 256), so that 3.5 times the tokens fit and a decode step
reads 3.5 times fewer cache bytes.

  * decode steps: ``rope_kv_append_int4`` and ``decode_attention_int4``;
  * prefill: the prompt's rows are appended, the context is read back in 16 bits
    (``kv_read_int4``) and runs through ``flash_attention_v2``: a prompt sees the
    same keys and values whether it comes in one piece or several.

The q/k/v projection with the append in its epilogue (``qkv_rope_append``)
writes 16-bit rows, so these caches turn it off for their steps: on 16-bit weights a
step of one short sequence takes 2% longer than with a 16-bit cache.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple, Union

import torch

from .flash_attention import flash_attention_v2
from .ops import (Int4KV, StepWorkspaces, decode_attention_int4, decode_attention_int4_workspace,
                  kv_read_int4, rope_kv_append_int4)
from .ragged_cache import RaggedKVCache

__all__ = ["Int4KVCache", "Int4RaggedKVCache"]


def _attend(kv: Int4KV, context: Optional[torch.Tensor], qkv: torch.Tensor, positions: torch.Tensor,
            ctx, num_heads: int, scale: float) -> torch.Tensor:
    """One layer's append and attention; ``context``: positions [B, end] of a
    prefill's keys."""
    B, S, _ = qkv.shape
    D = kv.head_dim
    q = rope_kv_append_int4(qkv, positions, ctx.cos_table, ctx.sin_table, kv, num_heads)
    if ctx.decode:
        out = decode_attention_int4(q.view(B, num_heads, D), kv, ctx.seq_lens, scale,
                                    workspace=ctx.workspace)
        return out.view(B, 1, num_heads * D)
    k, v = kv_read_int4(kv, context)
    out = flash_attention_v2(q, k, v, causal=True, sm_scale=scale)
    return out.transpose(1, 2).reshape(B, S, num_heads * D)


class Int4KVCache:
    """Dense 4-bit cache: ``KVCacheManager``'s constructor arguments, request
    lifecycle and step interface.  ``read`` gives a layer's rows in 16 bits (the
    counterpart of ``KVCacheManager.get``, as copies)."""

    def __init__(self, *, num_layers: int, max_batch_size: int, max_seq_len: int, n_kv_heads: int,
                 head_dim: int, dtype: torch.dtype = torch.float16,
                 device: Union[str, torch.device] = "cuda") -> None:
        if num_layers <= 0:
            raise ValueError("num_layers must be positive")
        if max_batch_size <= 0:
            raise ValueError("max_batch_size must be positive")
        if max_seq_len <= 0:
            raise ValueError("max_seq_len must be positive")
        if n_kv_heads <= 0 or head_dim <= 0:
            raise ValueError("n_kv_heads and head_dim must be positive")
        device = torch.device(device)
        if device.type != "cuda":
            raise RuntimeError("Int4KVCache lives in GPU memory: a CUDA device is required.")
        if not torch.cuda.is_available():
            raise RuntimeError("Int4KVCache requested CUDA but CUDA is unavailable.")
        self._setup([Int4KV.empty(max_batch_size, n_kv_heads, max_seq_len, head_dim, dtype, device)
                     for _ in range(num_layers)],
                    torch.zeros(max_batch_size, dtype=torch.int32, device=device))

    def _setup(self, layers: List[Int4KV], seq_lens: torch.Tensor) -> None:
        first = layers[0]
        self.layers, self.seq_lens = layers, seq_lens
        self.num_layers, self.max_batch_size = len(layers), first.max_batch
        self.max_seq_len, self.n_kv_heads = first.max_seq_len, first.kv_heads
        self.head_dim, self.dtype, self.device = first.head_dim, first.dtype, first.device
        self.active_batch_size = 0
        self._workspaces = StepWorkspaces()
        self._context: Optional[torch.Tensor] = None

    def row_view(self, start: int, count: int) -> "Int4KVCache":
        """Sequences ``[start, start + count)`` of this cache, in place."""
        view = Int4KVCache.__new__(Int4KVCache)
        view._setup([kv.rows(start, count) for kv in self.layers],
                    self.seq_lens[start:start + count])
        return view

    def memory_footprint_bytes(self) -> int:
        return sum(kv.memory_footprint_bytes() for kv in self.layers)

    # -- request lifecycle (kv_manager.py:170-204) --------------------------
    def begin_request(self, batch_size: int) -> None:
        if batch_size <= 0:
            raise ValueError("batch_size must be positive")
        if batch_size > self.max_batch_size:
            raise ValueError(f"batch_size={batch_size} exceeds max_batch_size={self.max_batch_size}")
        self.active_batch_size = batch_size
        self.seq_lens[:batch_size].zero_()

    def reset(self) -> None:
        if self.active_batch_size:
            self.seq_lens[: self.active_batch_size].zero_()
        self.active_batch_size = 0

    def current_seq_len(self, batch_idx: int = 0) -> int:
        if batch_idx < 0 or batch_idx >= self.max_batch_size:
            raise IndexError("invalid batch index")
        return int(self.seq_lens[batch_idx].item())

    def read(self, *, layer_idx: int, batch_size: int, seq_len: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """Rows ``[0, seq_len)`` of sequences ``[0, batch_size)`` in the cache's
        dtype, ``[B, Hkv, S, D]`` each."""
        if not 0 <= layer_idx < self.num_layers:
            raise IndexError("invalid layer index")
        if batch_size < 0 or seq_len < 0:
            raise ValueError("batch_size and seq_len must not be negative")
        if batch_size > self.max_batch_size:
            raise ValueError("batch size exceeds cache capacity")
        if seq_len > self.max_seq_len:
            raise ValueError("sequence length exceeds cache capacity")
        pos = torch.arange(seq_len, device=self.device).unsqueeze(0).expand(batch_size, -1)
        return kv_read_int4(self.layers[layer_idx], pos)

    # -- step interface used by the model -----------------------------------
    def decode_workspace(self, batch: int, num_heads: int) -> torch.Tensor:
        """Split partials of the decode kernel, kept across steps."""
        return self._workspaces.get((batch, num_heads), lambda: decode_attention_int4_workspace(
            self.layers[0], batch, num_heads))

    @torch.no_grad()
    def prepare_forward(self, positions: torch.Tensor, ctx, num_heads: int) -> None:
        B, S = positions.shape
        if B > self.max_batch_size:
            raise ValueError("batch size exceeds cache capacity")
        ctx.fused_qkv_max = 0
        if S == 1:
            ctx.decode = True
            self.seq_lens[:B].copy_(positions[:, -1] + 1)
            ctx.seq_lens = self.seq_lens[:B]
            ctx.workspace = self.decode_workspace(B, num_heads)
        else:
            ctx.decode = False
            ctx.start_pos = int(positions[0, 0].item())
            end = ctx.start_pos + S
            if end > self.max_seq_len:
                raise ValueError(f"KV cache overflow: end_pos={end}, max_seq_len={self.max_seq_len}")
            self._context = torch.arange(end, device=self.device).unsqueeze(0).expand(B, -1).contiguous()
            self.seq_lens[:B] = end

    def attend(self, *, layer_idx: int, positions: torch.Tensor, ctx, num_heads: int, scale: float,
               qkv: torch.Tensor) -> torch.Tensor:
        """RoPE + append of ``qkv`` [B, S, (H+2Hkv)*D], then causal attention of
        the new queries over the cached context; returns [B, S, H*D]."""
        if not 0 <= layer_idx < self.num_layers:
            raise IndexError(f"layer_idx={layer_idx} outside [0, {self.num_layers})")
        return _attend(self.layers[layer_idx], self._context, qkv, positions, ctx, num_heads, scale)


class Int4RaggedKVCache(RaggedKVCache):
    """``RaggedKVCache`` with 4-bit rows: the same constructor, selection of
    sequences and step interface."""

    def _allocate(self) -> None:
        self.layers = [Int4KV.empty_ragged(self.n_kv_heads, self.total_rows, self.head_dim,
                                           self.seq_base, self.seq_cap, self.max_seq_len, self.dtype,
                                           self.device) for _ in range(self.num_layers)]
        self._context: Optional[torch.Tensor] = None

    def memory_footprint_bytes(self) -> int:
        return sum(kv.memory_footprint_bytes() for kv in self.layers)

    def select(self, ids: Sequence[int]) -> None:
        super().select(ids)
        self.active = [kv.select(self.active_base, self.active_cap) for kv in self.layers]

    def decode_workspace(self, batch: int, num_heads: int) -> torch.Tensor:
        return self._workspaces.get((batch, num_heads), lambda: decode_attention_int4_workspace(
            self.layers[0], batch, num_heads))

    @torch.no_grad()
    def prepare_forward(self, positions: torch.Tensor, ctx, num_heads: int) -> None:
        super().prepare_forward(positions, ctx, num_heads)
        ctx.fused_qkv_max = 0
        if not ctx.decode:
            B, S = positions.shape
            end = ctx.start_pos + S
            self._context = torch.arange(end, device=self.device).unsqueeze(0).expand(B, -1).contiguous()

    def attend(self, *, layer_idx: int, positions: torch.Tensor, ctx, num_heads: int, scale: float,
               qkv: torch.Tensor) -> torch.Tensor:
        return _attend(self.active[layer_idx], self._context, qkv, positions, ctx, num_heads, scale)
