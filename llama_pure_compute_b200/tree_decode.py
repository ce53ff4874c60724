"""Speculative decoding: a drafted tree of tokens a sequence is verified in one forward.

The reference decodes one token a step (src/llama_pure_compute/generate.py:156-333).
Here a step runs the model on a tree of up to 64 tokens: its root is the token
sampled last, the others are a drafter's guesses of what follows.  The model draws
a token after every node; the branch that the draws agree with is kept, so that a
step yields one token more than it had right guesses.  What is generated has the
distribution of plain sampling whatever is drafted (the draw at a position has the
same random number in every tree), and is greedy decoding at temperature 0.

  * ``DraftTree``: the shape of the trees;
  * ``TreeCache``: the step interface of a ``KVCacheManager`` or ``RaggedKVCache``
    for a forward over trees (``rope_kv_append_tree``, ``tree_attention``);
  * ``BatchedTreeDecoder``: prefill, then steps replayed from one CUDA graph, with
    ``sample_tokens`` and ``tree_accept``.
"""
from __future__ import annotations

from typing import Callable, List, Optional, Sequence, Tuple, Union

import torch

from .generate import BatchedGreedyDecoder
from .kv_manager import KVCacheManager
from .ops import (MAX_TREE_NODES, LayerCaches, StepWorkspaces, decode_attention, decode_attention_ragged,
                  qkv_rope_append, rope_kv_append, rope_kv_append_ragged, rope_kv_append_tree,
                  sample_tokens, tree_accept, tree_attention, tree_attention_workspace)
from .ragged_cache import RaggedKVCache

__all__ = ["DraftTree", "TreeCache", "BatchedTreeDecoder"]


class DraftTree:
    """The shape of a drafted tree: ``parents[t]`` of node t, before it; -1 of the
    root, node 0.  ``parents`` and ``depths`` (int32 [T]) and ``masks`` (int64 [T],
    the bits of a node's ancestors and its own) are tensors on ``device``."""

    def __init__(self, parents: Sequence[int], device: Union[str, torch.device] = "cuda"):
        parents = [int(p) for p in parents]
        if not 1 <= len(parents) <= MAX_TREE_NODES:
            raise ValueError(f"a tree has 1 to {MAX_TREE_NODES} nodes")
        if parents[0] != -1 or any(not 0 <= p < t for t, p in enumerate(parents) if t):
            raise ValueError("parents must stand before their children, and only node 0 has none")
        depths, masks = [0], [1]
        for t in range(1, len(parents)):
            depths.append(depths[parents[t]] + 1)
            masks.append(masks[parents[t]] | 1 << t)
        self.nodes = len(parents)
        self.max_depth = max(depths)
        self.device = torch.device(device)
        self.parents = torch.tensor(parents, dtype=torch.int32, device=self.device)
        self.depths = torch.tensor(depths, dtype=torch.int32, device=self.device)
        self.masks = torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks],
                                  dtype=torch.int64, device=self.device)

    @classmethod
    def chain(cls, nodes: int, device: Union[str, torch.device] = "cuda") -> "DraftTree":
        """One branch: the root and ``nodes - 1`` tokens after it."""
        return cls(range(-1, nodes - 1), device)


class TreeCache:
    """A 16-bit cache for forwards over trees: ``LlamaForCausalLM`` takes it as its
    ``kv_cache`` with ``input_ids`` [B, T], row b a tree over the sequence of row b
    (a ragged cache's selection).  The nodes' K and V go to the rows behind the
    sequence's ``seq_lens`` keys; ``accept`` keeps a branch of them.  A tree of one
    node is a decode step, and takes that step's kernels."""

    def __init__(self, kv_cache: Union[KVCacheManager, RaggedKVCache], batch: int, tree: DraftTree):
        if type(kv_cache) not in (KVCacheManager, RaggedKVCache):
            raise TypeError("trees need a KVCacheManager or a RaggedKVCache")
        self.kv, self.batch, self.tree = kv_cache, batch, tree
        if tree.device.type != kv_cache.device.type or \
                (tree.parents.get_device() != kv_cache.seq_lens.get_device()):
            raise ValueError("the tree must be on the cache's device")
        if isinstance(kv_cache, RaggedKVCache):
            if batch != len(kv_cache.active_ids):
                raise ValueError(f"batch of {batch} rows but {len(kv_cache.active_ids)} selected "
                                 "sequences")
            # the selection of now: a captured step stays with it
            self._ids = kv_cache._idx
            self.base, self.cap = kv_cache.active_base, kv_cache.active_cap
            # the selection's lengths may be older than the sequences': as if selected again
            self.lens = kv_cache.active_lens = kv_cache.seq_lens[self._ids]
        else:
            if not 0 < batch <= kv_cache.max_batch_size:
                raise ValueError("batch size exceeds cache capacity")
            self.lens, self._ids = kv_cache.seq_lens[:batch], None
            self.base = self.cap = None
        if tree.nodes == 1:
            self.keys = torch.empty(batch, dtype=torch.int32, device=kv_cache.device)
            self.place = torch.empty(batch, 1, dtype=torch.int64, device=kv_cache.device)
        self.layers = LayerCaches(kv_cache.k_cache, kv_cache.v_cache, self.base, self.cap)
        self._workspaces = StepWorkspaces()

    # -- the model's step interface ---------------------------------------------
    @torch.no_grad()
    def prepare_forward(self, positions: torch.Tensor, ctx, num_heads: int) -> None:
        B, T = positions.shape
        if B != self.batch or T != self.tree.nodes:
            raise ValueError(f"forward of {B} x {T} tokens over {self.batch} trees of "
                             f"{self.tree.nodes} nodes")
        ctx.decode = True
        if self._ids is not None:  # where the sequences stand, whoever moved them
            with torch.inference_mode():  # the lengths may have been made there
                torch.index_select(self.kv.seq_lens, 0, self._ids, out=self.lens)
        if T == 1:
            self.place.copy_(self.lens[:, None])
            ctx.seq_lens = torch.add(self.lens, 1, out=self.keys)
            ctx.workspace = self.kv.decode_workspace(B, num_heads)
            return
        ctx.fused_qkv_max = 0  # that kernel's rows are its rotary positions
        ctx.seq_lens = self.lens
        ctx.workspace = None

    def attend(self, *, layer_idx: int, positions: torch.Tensor, ctx, num_heads: int, scale: float,
               qkv: Optional[torch.Tensor] = None, x: Optional[torch.Tensor] = None,
               packed_qkv=None, norm_eps: float = 0.0) -> torch.Tensor:
        kc, vc = self.kv.k_cache[layer_idx], self.kv.v_cache[layer_idx]
        if self.tree.nodes == 1:
            return self._attend_one(kc, vc, ctx, num_heads, scale, qkv, x, packed_qkv, norm_eps)
        q = rope_kv_append_tree(qkv, self.lens, self.tree.depths, ctx.cos_table, ctx.sin_table, kc,
                                vc, num_heads, self.kv.n_kv_heads, self.base, self.cap)
        if ctx.workspace is None:
            ctx.workspace = self._workspaces.get(q.shape, lambda: tree_attention_workspace(q, kc))
        out = tree_attention(q, kc, vc, self.lens, self.tree.masks, scale, self.base, self.cap,
                             ctx.workspace)
        B, H, T, D = out.shape
        return out.transpose(1, 2).reshape(B, T, H * D)  # a view: it is laid out so

    def _attend_one(self, kc, vc, ctx, num_heads, scale, qkv, x, packed_qkv, norm_eps):
        kv_heads, base, cap = self.kv.n_kv_heads, self.base, self.cap
        if packed_qkv is not None:
            q = qkv_rope_append(x, packed_qkv, self.place, ctx.cos_table, ctx.sin_table, kc, vc, num_heads,
                                kv_heads, seq_base=base, seq_cap=cap, norm_eps=norm_eps)
        elif base is None:
            q = rope_kv_append(qkv, self.place, ctx.cos_table, ctx.sin_table, kc, vc, num_heads, kv_heads)
        else:
            q = rope_kv_append_ragged(qkv, self.place, ctx.cos_table, ctx.sin_table, kc, vc, base, cap,
                                      num_heads, kv_heads)
        B, D = self.batch, self.kv.head_dim
        q = q.view(B, num_heads, D)
        if base is None:
            out = decode_attention(q, kc, vc, ctx.seq_lens, scale, workspace=ctx.workspace)
        else:
            out = decode_attention_ragged(q, kc, vc, ctx.seq_lens, base, cap, self.kv.max_seq_len, scale,
                                          workspace=ctx.workspace)
        return out.view(B, 1, num_heads * D)

    # -- after the forward --------------------------------------------------------
    @torch.no_grad()
    def accept(self, drafted: torch.Tensor, sampled: torch.Tensor, active: Optional[torch.Tensor] = None
               ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """``tree_accept`` in every layer; the sequences' lengths grow by what was
        accepted (times ``active``, int32 [B], if given: 0 leaves a sequence where it
        is, and its next root has to stay the one it had).  Returns (accepted, tokens,
        path), of a sequence that stays too what its tree would have given."""
        got = tree_accept(drafted, self.tree.parents, sampled, self.lens, self.layers)
        self.lens.add_(got[0] if active is None else got[0] * active)
        if self._ids is not None:
            self.kv.seq_lens.index_copy_(0, self._ids, self.lens)
        return got


class BatchedTreeDecoder(BatchedGreedyDecoder):
    """Speculative decoding of a (possibly ragged) batch, one graph replay a step.

    ``drafter(roots)`` gets the tokens sampled last (int64 [B], device) and returns
    its guesses for nodes 1 to T - 1 (int64 [B, T - 1]; one outside the vocabulary counts
    as its nearest token); it runs between the steps.
    ``temperature``, ``top_k``, ``top_p`` and ``min_p`` are those of
    ``sample_tokens`` (temperature 0: greedy), a number or a device tensor with one
    entry a sequence, which every step reads anew; ``generator`` makes the random
    numbers, one a sequence and position.  A token of -1: the model's logits left
    nothing to draw; the sequence goes on as after token 0.

    ``active`` (int32 [B], device; 1 after a prefill): a sequence whose entry is set to
    0 waits.  Steps leave its tokens and its length as they are and give 0 accepted
    tokens for it."""

    def __init__(self, model: torch.nn.Module, kv_cache: Union[KVCacheManager, RaggedKVCache],
                 batch_size: int, tree: DraftTree,
                 drafter: Optional[Callable[[torch.Tensor], torch.Tensor]] = None, *,
                 temperature: Union[float, torch.Tensor] = 0.0, top_k: Union[int, torch.Tensor] = 0,
                 top_p: Union[float, torch.Tensor] = 1.0, min_p: Union[float, torch.Tensor] = 0.0,
                 generator: Optional[torch.Generator] = None, use_cuda_graph: bool = True,
                 prefill_chunk: int = 16) -> None:
        if type(kv_cache) not in (KVCacheManager, RaggedKVCache):
            raise TypeError("trees need a KVCacheManager or a RaggedKVCache")
        super().__init__(model, kv_cache, batch_size, use_cuda_graph, prefill_chunk)
        if tree.nodes > 1 and drafter is None:
            raise ValueError("a tree of more than its root needs a drafter")
        self.tree, self.drafter = tree, drafter
        self.settings = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        for name, value in self.settings.items():
            if isinstance(value, torch.Tensor) and (value.get_device() != kv_cache.seq_lens.get_device()
                                                    or value.numel() != batch_size):
                raise ValueError(f"{name} must be a number or have one entry a sequence on the cache's device")
        self.generator = generator
        self.rows = model.config.max_seq_len  # of the rotary tables
        self.tokens = torch.zeros(batch_size, tree.nodes, dtype=torch.long, device=self.device)
        self.positions = torch.zeros(batch_size, tree.nodes, dtype=torch.long, device=self.device)
        self.active = torch.ones(batch_size, dtype=torch.int32, device=self.device)
        # a random number for the token at each position
        self.uniforms = torch.zeros(batch_size, self.rows + 1, device=self.device)
        self.accepted = torch.zeros(batch_size, dtype=torch.int32, device=self.device)
        self.new_tokens = torch.zeros(batch_size, tree.nodes, dtype=torch.long, device=self.device)
        self._none = torch.full((), -1, dtype=torch.long, device=self.device)
        self.cache: Optional[TreeCache] = None
        self.started = False  # a prefill's sequences stand where step() takes them on

    def _sample(self, logits: torch.Tensor, uniforms: torch.Tensor, start: int, stop: int) -> torch.Tensor:
        """Draws of sequences start to stop - 1, uniforms [stop - start, ...] each."""
        def of(value):
            if not isinstance(value, torch.Tensor):
                return value
            rows = value.reshape(-1)[start:stop]
            return rows.view(-1, *[1] * (uniforms.dim() - 1)).expand(uniforms.shape)
        return sample_tokens(logits, uniforms, **{name: of(value) for name, value in self.settings.items()})

    def _pick(self, logits: torch.Tensor, start: int, stop: int, length: int) -> torch.Tensor:
        return self._sample(logits, self.uniforms[start:stop, length], start, stop)

    @torch.inference_mode()
    def prefill(self, prompts: Union[torch.Tensor, List[List[int]]]) -> torch.Tensor:
        """Returns the first generated token of each sequence (device, [B])."""
        self.started = False
        self.uniforms.uniform_(generator=self.generator)
        first = super().prefill(prompts)
        self.active.fill_(1)
        if self.cache is None or self.graph is None:
            self.cache = TreeCache(self.kv, self.B, self.tree)
        elif self.ragged:  # the captured step has the lengths of its own selection
            self.cache.lens.copy_(self.kv.active_lens)
            self.kv.active_lens = self.cache.lens
        self.started = True
        return first

    def _begin(self, first: torch.Tensor, lens: List[int]) -> None:
        self.tokens[:, 0] = first.clamp(min=0)

    def _step_body(self) -> None:
        cache = self.cache
        torch.add(self.kv.seq_lens[:self.B, None], self.tree.depths, out=self.positions)
        logits = self.model(self.tokens, positions=self.positions, kv_cache=cache)
        # the token after a node stands one further
        u = self.uniforms.gather(1, (self.positions + 1).clamp_(max=self.rows))
        sampled = self._sample(logits, u, 0, self.B)
        accepted, tokens, _ = cache.accept(self.tokens, sampled, self.active)
        goes = self.active[:, None] != 0
        had = self.tokens[:, :1]
        roots = tokens.gather(1, (accepted[:, None] - 1).long()).clamp_(min=0)
        torch.where(goes, roots, had, out=had)
        torch.mul(accepted, self.active, out=self.accepted)
        torch.where(goes, tokens, self._none, out=self.new_tokens)

    @torch.inference_mode()
    def capture(self) -> None:
        if not self.started:
            raise RuntimeError("prefill first")
        lens = self.kv.seq_lens[:self.B]
        lens0 = lens.clone()
        tok0 = self.tokens.clone()
        s = torch.cuda.Stream(self.device)
        s.wait_stream(torch.cuda.current_stream(self.device))
        with torch.cuda.stream(s):
            self._step_body()
        torch.cuda.current_stream(self.device).wait_stream(s)
        for t in (lens, self.cache.lens):
            t.copy_(lens0)
        self.tokens.copy_(tok0)
        torch.cuda.synchronize(self.device)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            self._step_body()
        self.graph = g
        torch.cuda.synchronize(self.device)

    @torch.inference_mode()
    def step(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """One forward: (tokens [B, T], accepted [B]) on the device -- sequence b goes on
        by ``tokens[b, :accepted[b]]``.  Its cache needs T free rows.  After ``generate``,
        whose sequences end at different steps, and after a prefill that failed, a prefill
        comes first."""
        if not self.started:
            raise RuntimeError("prefill first")
        if self.tree.nodes > 1:
            guesses = self.drafter(self.tokens[:, 0].clone())
            if guesses.shape != (self.B, self.tree.nodes - 1) or guesses.dtype != torch.int64:
                raise ValueError(f"the drafter gave {tuple(guesses.shape)} {guesses.dtype}, not int64 "
                                 f"{(self.B, self.tree.nodes - 1)}")
            self.tokens[:, 1:].copy_(guesses.clamp(0, self.model.config.vocab_size - 1))
        if self.use_graph:
            if self.graph is None:
                self.capture()
            self.graph.replay()
        else:
            self._step_body()
        return self.new_tokens, self.accepted

    @torch.inference_mode()
    def generate(self, prompts, max_new_tokens: int) -> torch.Tensor:
        """Prefill and steps until every sequence has ``max_new_tokens``; [B,
        max_new_tokens] ids (device).  Reads the accepted counts after each step."""
        rows = prompts if isinstance(prompts, torch.Tensor) else list(prompts)
        caps = self.kv.capacities[:self.B] if self.ragged else [self.kv.max_seq_len] * self.B
        for r, cap in zip(rows, caps):
            # the last step may overshoot by a branch, and the sequence goes along, unchanged,
            # until the others are done
            most = len(r) + max_new_tokens - 1 + self.tree.max_depth
            if most + self.tree.nodes > cap:
                raise ValueError(f"a prompt of {len(r)} and {max_new_tokens} new tokens need "
                                 f"{most + self.tree.nodes} rows with these trees; the cache has {cap}")
            if most + self.tree.max_depth >= self.rows:
                raise ValueError("Requested generation exceeds configured max_seq_len.")
        out = torch.empty(self.B, max_new_tokens, dtype=torch.long, device=self.device)
        out[:, 0] = self.prefill(rows)
        have = [1] * self.B
        try:
            while min(have) < max_new_tokens:
                tokens, accepted = self.step()
                for b, n in enumerate(accepted.tolist()):
                    if have[b] < max_new_tokens:
                        n = min(n, max_new_tokens - have[b])
                        out[b, have[b]:have[b] + n] = tokens[b, :n]
                        have[b] += n
                self.active.copy_(torch.tensor([int(h < max_new_tokens) for h in have], dtype=torch.int32))
        finally:
            self.started = False
        return out
