"""Oracle of the 4-bit cache and weights: the formats' definitions, in fp32 where
the definition names fp32 roundings and in 64 bits everywhere else."""
from __future__ import annotations

import torch


def quantize_rows_ref(x: torch.Tensor):
    """Cache rows of x [..., D] (bf16/fp16): codes uint8 [..., D/2] (dim j low,
    dim j + D/2 high) and numbers [..., 4] = (s0, m0, s1, m1), every fp32
    operation rounded once."""
    D = x.shape[-1]
    g = x.float().reshape(*x.shape[:-1], 2, D // 2)
    lo, hi = g.amin(-1), g.amax(-1)  # NaN propagates
    s = ((hi - lo) / 15.0).to(x.dtype)
    sf = s.float()
    bad = ~(sf < float("inf"))
    tiny = ~bad & (sf < 2.0 ** -126)
    inv = torch.where(bad | tiny | (sf == 0), torch.zeros_like(sf), 1.0 / sf)
    c = torch.round((g - lo[..., None]) * inv[..., None]).clamp(0, 15)
    c = torch.where((bad | tiny)[..., None], torch.zeros_like(c), c)
    c = torch.nan_to_num(c, nan=0.0).to(torch.uint8)
    nan = torch.full_like(s, float("nan"))
    s = torch.where(bad, nan, torch.where(tiny, torch.zeros_like(s), s))
    m = torch.where(bad, nan, lo.to(x.dtype))
    numbers = torch.stack([s[..., 0], m[..., 0], s[..., 1], m[..., 1]], -1)
    return c[..., 0, :] | (c[..., 1, :] << 4), numbers


def rows_ref(codes: torch.Tensor, numbers: torch.Tensor) -> torch.Tensor:
    """The values of cache rows, in 64 bits."""
    n = numbers.double()
    return torch.cat([(codes & 15).double() * n[..., 0:1] + n[..., 1:2],
                      (codes >> 4).double() * n[..., 2:3] + n[..., 3:4]], -1)


def attention_ref(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float):
    """One sequence: q [H, D], k and v [Hkv, L, D] -> (out [H, D], the sum of
    p |v| behind each output), in 64 bits; zeros for L = 0."""
    H, D = q.shape
    Hkv, L, _ = k.shape
    if L == 0:
        z = torch.zeros(H, D, dtype=torch.float64, device=q.device)
        return z, z
    p = torch.softmax(q.double().view(Hkv, H // Hkv, D) @ k.double().mT * scale, -1)
    return (p @ v.double()).view(H, D), (p @ v.double().abs()).view(H, D)


def weight_ref(codes: torch.Tensor, scales: torch.Tensor, mins: torch.Tensor) -> torch.Tensor:
    """[rows, k] values of a 4-bit weight (column 2j low, 2j + 1 high), in 64 bits."""
    rows, ng = scales.shape
    c = torch.stack([codes & 15, codes >> 4], -1).double().reshape(rows, ng, -1)
    return (c * scales.double()[..., None] + mins.double()[..., None]).reshape(rows, -1)
