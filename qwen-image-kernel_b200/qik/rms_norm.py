"""Residual addition + RMS norm of a transformer decoder, next to the layer norms of
``qik.triton_fused`` (the reference has no such operator).

One call takes the sublayer's output ``x`` and the residual stream, and returns the new
stream ``x + residual`` and its RMS norm, either in the tensors' type or already as the
e4m3 codes and scale of the FP8 linear that follows (``FP8Linear.forward_e4m3``):

    h = x + residual                                        (fp32, stored rounded once)
    y = h * rsqrt(mean(h ** 2) + eps) * weight              (from the unrounded h)
    scale = max(max|y| / 448, 1e-12);  codes = e4m3(y / scale)

bf16 and fp16; the kernels are in ``csrc/qik_norm.cu``.
"""
from __future__ import annotations

import torch

from . import _lib as L

_TYPES = (torch.bfloat16, torch.float16)


def _row_pitch(t: torch.Tensor, M: int, N: int) -> tuple[torch.Tensor, int]:
    """t ([..., N]) and its row pitch in elements, copied only where the leading dims do
    not flatten to rows of one pitch or the alignment is not 16 bytes."""
    if t.is_contiguous():
        if t.data_ptr() % 16 == 0:
            return t, N
        return t.clone(), N
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= N and t.stride(0) % 8 == 0 and t.data_ptr() % 16 == 0:
        return t, t.stride(0)
    return t.contiguous(), N


def _check(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, who: str) -> tuple[int, int]:
    if not x.is_cuda:
        raise ValueError(f"qik: {who}: x must be a CUDA tensor (the kernels have no CPU path)")
    if x.dtype not in _TYPES:
        raise TypeError(f"qik: {who}: bf16 or fp16, got {x.dtype}")
    if x.dim() == 0:
        raise ValueError(f"qik: {who}: x needs at least one dimension")
    N = x.shape[-1]
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"qik: {who}: residual {tuple(residual.shape)} {residual.dtype} on {residual.device} does not "
                         f"match x {tuple(x.shape)} {x.dtype} on {x.device}")
    if weight.dim() != 1 or weight.shape[0] != N or weight.device != x.device:
        raise ValueError(f"qik: {who}: weight has shape {tuple(weight.shape)} on {weight.device}, expected ({N},) on "
                         f"{x.device}")
    if weight.dtype != x.dtype and weight.dtype != torch.float32:
        raise TypeError(f"qik: {who}: weight must be {x.dtype} or fp32, got {weight.dtype}")
    if N == 0 or N % 8 or N > 32768:
        raise ValueError(f"qik: {who}: {N} columns (a multiple of 8, at most 32768)")
    return x.numel() // N, N


def _weight(weight: torch.Tensor) -> torch.Tensor:
    return weight if weight.stride(0) == 1 and weight.data_ptr() % 16 == 0 else weight.clone(
        memory_format=torch.contiguous_format)


def fused_add_rms_norm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor,
                       eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """x, residual: [..., N] bf16 or fp16 (residual None: the plain norm of x); weight [N] of
    the same type or fp32.  Returns (norm, x + residual), both contiguous in x's type;
    the second is x itself without a residual."""
    M, N = _check(x, residual, weight, "fused_add_rms_norm")
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    h = x if residual is None else torch.empty_like(y)
    if M == 0:
        return y, h
    w = _weight(weight)
    xr, ldx = _row_pitch(x, M, N)
    rr, ldr = (None, 0) if residual is None else _row_pitch(residual, M, N)
    L.launch("qik_add_rms_norm", x.device, xr.data_ptr(), ldx, None if rr is None else rr.data_ptr(), ldr, w.data_ptr(),
             w.dtype == torch.float32, M, N, eps, x.dtype == torch.float16,
             None if residual is None else h.data_ptr(), y.data_ptr())
    return y, h


def fused_add_rms_norm_e4m3(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float,
                            scales: str = "tensor") -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """As ``fused_add_rms_norm`` with the norm quantized: returns (codes e4m3 [..., N],
    scale fp32, x + residual).  ``scales="tensor"``: one scale, shape [1], which
    ``FP8Linear.forward_e4m3`` takes; ``scales="row"``: one for each row, shape [...]."""
    M, N = _check(x, residual, weight, "fused_add_rms_norm_e4m3")
    if scales not in ("tensor", "row"):
        raise ValueError(f"qik: fused_add_rms_norm_e4m3: scales is 'tensor' or 'row', got {scales!r}")
    by_row = scales == "row"
    dev = x.device
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=dev)
    h = x if residual is None else torch.empty(x.shape, dtype=x.dtype, device=dev)
    s = torch.empty(x.shape[:-1] if by_row else 1, dtype=torch.float32, device=dev)
    if M == 0:
        if not by_row:
            s.fill_(1e-12)
        return q, s, h
    w = _weight(weight)
    xr, ldx = _row_pitch(x, M, N)
    rr, ldr = (None, 0) if residual is None else _row_pitch(residual, M, N)
    ws = None if by_row else torch.empty(L.load().qik_add_rms_norm_workspace_bytes(M), dtype=torch.uint8, device=dev)
    L.launch("qik_add_rms_norm_e4m3", dev, xr.data_ptr(), ldx, None if rr is None else rr.data_ptr(), ldr, w.data_ptr(),
             w.dtype == torch.float32, M, N, eps, x.dtype == torch.float16,
             None if residual is None else h.data_ptr(), q.data_ptr(), s.data_ptr(), by_row,
             None if ws is None else ws.data_ptr())
    return q, s, h
