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


_one: dict = {}  # a scale's shape and type on each device, for empty_like


def _row_pitch(t: torch.Tensor, N: int) -> tuple[torch.Tensor, int]:
    """t ([..., N]) and its row pitch in elements, copied only where the leading dims do
    not flatten to rows of one pitch or the alignment is not 16 bytes."""
    if t.is_contiguous():
        return (t, N) if t.data_ptr() % 16 == 0 else (t.clone(), N)
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= N and t.stride(0) % 8 == 0 and t.data_ptr() % 16 == 0:
        return t, t.stride(0)
    return t.contiguous(), N


def _prepare(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, who: str) -> tuple:
    """(x, its pitch, the residual's address and pitch, weight, whether it is fp32, rows,
    columns), checked; and the tensors that have to live until the launch."""
    if not x.is_cuda:
        raise ValueError(f"qik: {who}: x must be a CUDA tensor (the kernels have no CPU path)")
    dtype, shape, dev = x.dtype, x.shape, x.device
    if dtype not in _TYPES:
        raise TypeError(f"qik: {who}: bf16 or fp16, got {dtype}")
    if not shape:
        raise ValueError(f"qik: {who}: x needs at least one dimension")
    N = shape[-1]
    if N == 0 or N % 8 or N > 32768:
        raise ValueError(f"qik: {who}: {N} columns (a multiple of 8, at most 32768)")
    if weight.shape != (N,) or weight.device != dev:
        raise ValueError(f"qik: {who}: weight has shape {tuple(weight.shape)} on {weight.device}, expected ({N},) on {dev}")
    f32 = weight.dtype == torch.float32
    if not f32 and weight.dtype != dtype:
        raise TypeError(f"qik: {who}: weight must be {dtype} or fp32, got {weight.dtype}")
    if not weight.is_contiguous() or weight.data_ptr() % 16:
        weight = weight.clone(memory_format=torch.contiguous_format)
    x, ldx = _row_pitch(x, N)
    if residual is None:
        return x, ldx, None, 0, weight, f32, x.numel() // N, N, None
    if residual.shape != shape or residual.dtype != dtype or residual.device != dev:
        raise ValueError(f"qik: {who}: residual {tuple(residual.shape)} {residual.dtype} on {residual.device} does not "
                         f"match x {tuple(shape)} {dtype} on {dev}")
    residual, ldr = _row_pitch(residual, N)
    return x, ldx, residual.data_ptr(), ldr, weight, f32, x.numel() // N, N, residual


def fused_add_rms_norm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor,
                       eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """x, residual: [..., N] bf16 or fp16 (residual None: the plain norm of x); weight [N] of
    the same type or fp32.  Returns (norm, x + residual), both contiguous in x's type;
    the second is x itself without a residual."""
    xr, ldx, r, ldr, w, f32, M, N, keep = _prepare(x, residual, weight, "fused_add_rms_norm")
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    h = x if r is None else torch.empty_like(y)
    if M:
        L.launch("qik_add_rms_norm", x.device.index, xr.data_ptr(), ldx, r, ldr, w.data_ptr(), f32, M, N, eps,
                 x.dtype == torch.float16, None if r is None else h.data_ptr(), y.data_ptr())
    return y, h


def fused_add_rms_norm_e4m3(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float,
                            scales: str = "tensor") -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """As ``fused_add_rms_norm`` with the norm quantized: returns (codes e4m3 [..., N],
    scale fp32, x + residual).  ``scales="tensor"``: one scale, shape [1], which
    ``FP8Linear.forward_e4m3`` takes; ``scales="row"``: one for each row, shape [...]."""
    xr, ldx, r, ldr, w, f32, M, N, keep = _prepare(x, residual, weight, "fused_add_rms_norm_e4m3")
    idx = x.device.index
    q = torch.empty_like(x, dtype=torch.float8_e4m3fn, memory_format=torch.contiguous_format)
    h = x if r is None else torch.empty_like(x, memory_format=torch.contiguous_format)
    ws, by_row = None, scales == "row"
    if by_row:
        s = x.new_empty(x.shape[:-1], dtype=torch.float32)
    elif scales == "tensor":
        one = _one.get(idx)
        if one is None:
            one = _one[idx] = torch.empty(1, dtype=torch.float32, device=x.device)
        s = torch.empty_like(one)
        if M == 0:
            s.fill_(1e-12)
        else:
            n = L.on_device("qik_add_rms_norm_workspace_bytes", idx, M, N)
            ws = x.new_empty(n, dtype=torch.uint8) if n else None
    else:
        raise ValueError(f"qik: fused_add_rms_norm_e4m3: scales is 'tensor' or 'row', got {scales!r}")
    if M:
        L.launch("qik_add_rms_norm_e4m3", idx, xr.data_ptr(), ldx, r, ldr, w.data_ptr(), f32, M, N, eps,
                 x.dtype == torch.float16, None if r is None else h.data_ptr(), q.data_ptr(), s.data_ptr(), by_row,
                 None if ws is None else ws.data_ptr())
    return q, s, h
