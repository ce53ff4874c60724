"""Decode-step projections on 4-bit weights with group scales (``lpc_int4_pack`` +
``lpc_int4_linear``), the 4-bit sibling of ``packed_linear``.

A decode step of a few sequences only streams weights, so its time goes with
their bytes: 4-bit codes with a scale and a minimum per group of 128 columns
take 0.53 bytes a weight, against 2.  ``Int4Weight`` owns the packed bytes;
``int4_linear`` runs one product with its epilogue (residual add, SiLU * up).
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from .ops import _dense16, _overlap, _require_cuda

__all__ = ["Int4Weight", "int4_linear", "MAX_TOKENS"]

EPILOGUES = {"store": 0, "residual": 1, "swiglu": 2}
LAYOUTS = {"linear": 0, "swiglu": 1}
MAX_TOKENS = 64


class Int4Weight:
    """A weight in 4 bits: column k of row n stands for
    ``scales[n, g] * c + mins[n, g]``, c in 0..15, g = k // group_size
    (32, 64 or 128 columns).

    ``Int4Weight(w0, w1)`` quantises a bf16 or fp16 weight: per row and group
    ``m = min``, ``s = (max - m) / 15``, codes rounded to nearest.
    layout "linear": ``w0`` is ``[n_out, k]``.
    layout "swiglu": ``w0`` holds the gate rows ``[n_out, k]`` and ``w1`` the up
    rows, or ``w1`` is None and ``w0`` is the fused ``[2 n_out, k]`` weight.

    ``Int4Weight.from_codes`` takes a weight that is in 4 bits already.
    k must be a multiple of 64 and of ``group_size``.
    """

    def __init__(self, w0: torch.Tensor, w1: Optional[torch.Tensor] = None,
                 layout: str = "linear", group_size: int = 128):
        if layout not in LAYOUTS:
            raise ValueError(f"LlamaPureComputeError: unknown packed layout {layout!r}")
        for t in (w0,) if w1 is None else (w0, w1):
            self._check_source(t)
            if t.shape[1] != w0.shape[1]:
                raise ValueError("LlamaPureComputeError: weights must be 2-D, of the same width.")
            if t.dtype != w0.dtype or t.device != w0.device:
                raise ValueError("LlamaPureComputeError: up weight must match the gate weight.")
        if w1 is not None and (layout != "swiglu" or w1.shape != w0.shape):
            raise ValueError("LlamaPureComputeError: up weight must match the gate weight (layout "
                             "'swiglu').")
        k = w0.shape[1]
        self._check_sizes(k, group_size)
        parts = [self.quantize(t.detach(), group_size) for t in ((w0,) if w1 is None else (w0, w1))]
        codes, scales, mins = (torch.cat(p) if len(p) > 1 else p[0] for p in zip(*parts))
        self._pack(codes, scales, mins, layout, group_size)

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor, mins: torch.Tensor, *,
                   group_size: int, layout: str = "linear") -> "Int4Weight":
        """codes uint8 ``[rows, k/2]`` (column 2j in the low, 2j + 1 in the high
        four bits of byte j), scales and mins (bf16 or fp16)
        ``[rows, k/group_size]``; layout "swiglu": gate rows first, then up rows."""
        if layout not in LAYOUTS:
            raise ValueError(f"LlamaPureComputeError: unknown packed layout {layout!r}")
        for t, n in ((codes, "codes"), (scales, "scales"), (mins, "mins")):
            _require_cuda(t, n)
            if t.dim() != 2 or t.device != codes.device:
                raise ValueError("LlamaPureComputeError: codes, scales and mins must be 2-D on one "
                                 "device.")
        if codes.dtype != torch.uint8:
            raise TypeError("LlamaPureComputeError: codes must be uint8.")
        if scales.dtype not in (torch.bfloat16, torch.float16) or mins.dtype != scales.dtype:
            raise TypeError("LlamaPureComputeError: scales and mins must be bf16 or fp16, both alike.")
        rows, k = codes.shape[0], 2 * codes.shape[1]
        cls._check_sizes(k, group_size)
        if tuple(scales.shape) != (rows, k // group_size) or mins.shape != scales.shape:
            raise ValueError("LlamaPureComputeError: scales and mins must be [rows, k / group_size].")
        self = cls.__new__(cls)
        self._pack(codes, scales, mins, layout, group_size)
        return self

    @classmethod
    def check(cls, w: torch.Tensor, group_size: int = 128) -> None:
        """Raises what ``Int4Weight(w, group_size=)`` would of its arguments and
        values, and makes nothing."""
        cls._check_source(w)
        cls._check_sizes(w.shape[1], group_size)
        for _ in cls._stretches(w.detach(), group_size):
            pass

    @staticmethod
    def _check_source(w: torch.Tensor) -> None:
        _require_cuda(w, "weight")
        if w.dim() != 2:
            raise ValueError("LlamaPureComputeError: weights must be 2-D, of the same width.")
        if w.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError("LlamaPureComputeError: int4 weights are made of bf16 or fp16 weights.")

    @staticmethod
    def _check_sizes(k: int, group_size: int) -> None:
        if group_size not in (32, 64, 128):
            raise ValueError("LlamaPureComputeError: group_size must be 32, 64 or 128.")
        if k == 0 or k % 64 or k % group_size:
            raise ValueError(f"LlamaPureComputeError: k = {k} must be a multiple of 64 and of "
                             f"group_size ({group_size}).")

    @staticmethod
    def quantize(w: torch.Tensor, group_size: int = 128):
        """(codes, scales, mins) of a ``[rows, k]`` weight, as ``from_codes``
        takes them; runs where the weight is, a stretch of rows at a time."""
        rows, k = w.shape
        Int4Weight._check_sizes(k, group_size)
        codes = torch.empty(rows, k // 2, dtype=torch.uint8, device=w.device)
        scales = torch.empty(rows, k // group_size, dtype=w.dtype, device=w.device)
        mins = torch.empty_like(scales)
        for at, g, lo, s in Int4Weight._stretches(w, group_size):
            sf = s.float()[..., None]
            c = ((g - lo[..., None]) / torch.where(sf == 0, torch.ones_like(sf), sf)).round_()
            c = c.clamp_(0, 15).to(torch.uint8).view(-1, k // 2, 2)
            to = slice(at, at + c.shape[0])
            codes[to] = c[..., 0] | (c[..., 1] << 4)
            scales[to], mins[to] = s, lo.to(w.dtype)
        return codes, scales, mins

    @staticmethod
    def _stretches(w: torch.Tensor, group_size: int):
        """(first row, groups in fp32, their minima in fp32, their scales in w's
        dtype) of some rows at a time."""
        k = w.shape[1]
        step = max(1, (1 << 25) // k)
        for at in range(0, w.shape[0], step):
            g = w[at:at + step].float().view(-1, k // group_size, group_size)
            lo, hi = g.amin(-1), g.amax(-1)
            if not bool((lo.isfinite() & hi.isfinite()).all()):
                raise ValueError("LlamaPureComputeError: a weight with non-finite values has no 4-bit form.")
            s = ((hi - lo) / 15).to(w.dtype)
            if not bool(s.isfinite().all()):
                raise ValueError("LlamaPureComputeError: a group's range overflows the scale's dtype.")
            yield at, g, lo, s

    def _pack(self, codes, scales, mins, layout, group_size) -> None:
        rows = codes.shape[0]
        if layout == "swiglu" and rows % 2:
            raise ValueError("LlamaPureComputeError: fused gate/up weight needs an even row count.")
        self.n_out = rows // 2 if layout == "swiglu" else rows
        self.k, self.layout, self.group_size = 2 * codes.shape[1], layout, group_size
        self.dtype, self.device = scales.dtype, codes.device
        lib = _lib.load()
        lay = LAYOUTS[layout]
        nbytes = lib.lpc_int4_weight_bytes(self.n_out, self.k, group_size, lay)
        if nbytes <= 0:
            raise ValueError(f"LlamaPureComputeError: cannot pack a [{rows}, {self.k}] weight.")
        self.data = torch.empty(nbytes, dtype=torch.uint8, device=codes.device)
        self._c = _lib.W4(self.data.data_ptr(), self.n_out, self.k, group_size, lay,
                          _lib.DTYPE_CODE[self.dtype])
        self.ref = ctypes.addressof(self._c)
        self._workspace = {}  # tokens -> bytes
        self._linear = lib.lpc_int4_linear
        codes, scales, mins = codes.contiguous(), scales.contiguous(), mins.contiguous()
        self.index = codes.get_device()
        rc = _lib.call_on(self.index, lib.lpc_int4_pack, self.ref, codes.data_ptr(),
                          scales.data_ptr(), mins.data_ptr())
        _lib.check(rc, "int4_pack")
        _lib.count_launch("lpc_int4_pack")

    def memory_footprint_bytes(self) -> int:
        return self.data.numel()

    def workspace_bytes(self, tokens: int) -> int:
        """Scratch that a product of this many tokens takes from torch's allocator."""
        n = self._workspace.get(tokens)
        if n is None:
            n = _lib.load().lpc_int4_linear_workspace_bytes(self.ref, tokens)
            self._workspace[tokens] = n
        return n

    def dequantize(self) -> torch.Tensor:
        """The 16-bit weight that the codes stand for, ``[n_out, k]`` (layout
        "swiglu": ``[2 n_out, k]``, gate rows first): for token counts beyond
        ``MAX_TOKENS``, whose products are library GEMMs.  Writing the copy and reading
        it back costs several times a decode-sized GEMM."""
        rows = self.n_out * (2 if self.layout == "swiglu" else 1)
        out = torch.empty(rows, self.k, dtype=self.dtype, device=self.device)
        rc = _lib.call_on(self.index, _lib.load().lpc_int4_unpack, self.ref, out.data_ptr())
        _lib.check(rc, "int4_unpack")
        _lib.count_launch("lpc_int4_unpack")
        return out


def int4_linear(x: torch.Tensor, w: Int4Weight, epilogue: str = "store",
                resid: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``epilogue(x w^T)`` for ``x [..., k]`` with at most 64 rows.

    "store": x w^T.  "residual": resid + x w^T (``out`` may be ``resid``).
    "swiglu": silu(x Wg^T) * (x Wu^T) on a weight of layout "swiglu".
    Sums in fp32, rounded once to x's dtype.  Larger products (about n k > 18 * 2^20
    from 17 rows on, 8 * 2^20 from 33, 4.5 * 2^20 from 49; 72 * 2^20 for fewer rows
    that do not fit shared memory) round each weight ``s c + m`` to fp16's 11 bits first,
    as a 16-bit copy of the weight would: bf16 results do not show it, fp16 ones are
    2.9e-4 off in the mean instead of 2.1e-4 (SwiGLU 3.5e-4; 5e-4 where x is of one
    sign).
    """
    epi = EPILOGUES.get(epilogue)
    if epi is None:
        raise ValueError(f"LlamaPureComputeError: unknown epilogue {epilogue!r}")
    if (epi == 2) != (w.layout == "swiglu"):
        raise ValueError("LlamaPureComputeError: the swiglu epilogue needs a swiglu-packed weight.")
    index, n, k, shape = w.index, w.n_out, w.k, x.shape
    if x.get_device() != index or not shape or shape[-1] != k or x.dtype != w.dtype:
        _require_cuda(x, "x")
        raise ValueError("LlamaPureComputeError: x must be [..., k] in the weight's dtype and device.")
    tokens = shape[0] if len(shape) == 2 else x.numel() // k
    if tokens > MAX_TOKENS:
        raise ValueError(f"LlamaPureComputeError: int4_linear takes at most {MAX_TOKENS} rows.")
    xp = x.data_ptr()
    if xp % 16 or not x.is_contiguous():
        x = _dense16(x)
        xp = x.data_ptr()
    rp = None
    if epi == 1:
        if resid is None or resid.numel() != tokens * n or not resid.dim() or resid.shape[-1] != n \
                or not resid.is_contiguous() or resid.dtype != x.dtype or resid.get_device() != index:
            raise ValueError("LlamaPureComputeError: residual must be a contiguous [..., n_out] tensor.")
        rp = resid.data_ptr()
    elif resid is not None:
        raise ValueError("LlamaPureComputeError: resid is for the residual epilogue.")
    if out is None:
        out = x.new_empty(tokens, n) if len(shape) == 2 else x.new_empty(*shape[:-1], n)
    elif out.numel() != tokens * n or not out.dim() or out.shape[-1] != n or not out.is_contiguous() \
            or out.dtype != x.dtype or out.get_device() != index:
        raise ValueError("LlamaPureComputeError: out must be a contiguous [..., n_out] tensor.")
    elif _overlap(out, x):
        raise ValueError("LlamaPureComputeError: out must not be x or overlap it.")
    elif rp is not None and out.data_ptr() != rp and _overlap(out, resid):
        raise ValueError("LlamaPureComputeError: out may be resid, but not overlap it otherwise.")
    if not tokens:
        return out
    need = w._workspace.get(tokens)
    if need is None:
        need = w.workspace_bytes(tokens)
    ws = x.new_empty((need + 1) // 2) if need else None
    rc = _lib.call_on(index, w._linear, w.ref, xp, out.data_ptr(), rp, tokens, epi,
                      ws.data_ptr() if need else None, need)
    if rc:
        _lib.check(rc, "int4_linear")
    _lib.launch_count += 2 if need else 1
    return out
