"""Plain definitions, in 64 bits, of the operators of a speculative decoding step over drafted
trees: sampling with filters, attention of a tree over its context, acceptance of a branch."""
import math
from typing import List, Sequence, Tuple

import torch


def sample_ref(logits: torch.Tensor, u: float, temperature: float = 1.0, top_k: int = 0,
               top_p: float = 1.0, min_p: float = 0.0) -> int:
    """The token of one row (see ``ops.sample_tokens``)."""
    x = logits.detach().cpu().double()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    order = torch.argsort(-x, stable=True)
    order = order[x[order] > -math.inf]
    if not order.numel():
        return -1
    if temperature == 0:
        return int(order[0])
    top = x[order[0]]
    xs = x[order]
    w = torch.exp(torch.where(xs == top, torch.zeros_like(xs), xs - top) / temperature)
    if 0 < top_k < order.numel():
        order, w = order[:top_k], w[:top_k]
    if top_p < 1:
        before = torch.cat([torch.zeros(1, dtype=w.dtype), torch.cumsum(w, 0)[:-1]])
        n = int((before <= top_p * w.sum()).sum())
        order, w = order[:n], w[:n]
    order, by = order[w >= min_p].sort()
    run = torch.cumsum(w[w >= min_p][by], 0)
    at = int((run <= u * run[-1]).sum())
    return int(order[min(at, order.numel() - 1)])


def tree_masks_ref(parents: Sequence[int]) -> Tuple[List[int], List[int]]:
    """(ancestors and self as bits, signed 64-bit; depth) of each node."""
    masks, depths = [], []
    for t, p in enumerate(parents):
        masks.append((masks[p] if p >= 0 else 0) | 1 << t)
        depths.append(depths[p] + 1 if p >= 0 else 0)
    return [m - (1 << 64) if m >> 63 else m for m in masks], depths


def tree_attention_ref(q, k, v, n: int, masks, scale: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """One sequence: q [H, T, D], k and v [Hkv, >= n + T, D] (rows of the cache), masks int64 [T].
    Returns the output [H, T, D] and the same with |v| for v, which bounds what a relative error
    of the weights does to it.  Rows that a node does not see take no part, whatever they hold."""
    heads, nodes, dim = q.shape
    kv = k.shape[0]
    out = torch.zeros(2, heads, nodes, dim, dtype=torch.float64, device=q.device)
    q, k, v = q.double().view(kv, heads // kv, nodes, dim), k.double(), v.double()
    masks = [int(m) for m in masks]
    for t in range(nodes):
        rows = list(range(n)) + [n + i for i in range(nodes) if masks[t] >> i & 1]
        if rows:
            s = torch.einsum("hgd,hrd->hgr", q[:, :, t], k[:, rows]) * scale
            p = torch.softmax(s, -1)
            for o, x in zip(out, (v, v.abs())):
                o[:, t] = torch.einsum("hgr,hrd->hgd", p, x[:, rows]).reshape(heads, dim)
    return out[0], out[1]


def accept_ref(drafted: Sequence[int], parents: Sequence[int], sampled: Sequence[int]):
    """(path, tokens) of one tree."""
    path = [0]
    while True:
        nxt = [c for c in range(1, len(drafted))
               if parents[c] == path[-1] and parents[c] < c and drafted[c] == sampled[path[-1]]]
        if not nxt:
            return path, [sampled[t] for t in path]
        path.append(nxt[0])
