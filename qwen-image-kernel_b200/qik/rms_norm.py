"""Residual addition + RMS norm of a transformer decoder, next to the layer norms of
``qik.triton_fused`` (the reference has no such operator).

One call takes the sublayer's output ``x`` and the residual stream, and returns the new
stream ``x + residual`` and its RMS norm, either in the tensors' type or already as the
e4m3 codes and scale of the FP8 linear that follows (``FP8Linear.forward_e4m3``):

    h = x + residual                                        (fp32, stored rounded once)
    y = h * rsqrt(mean(h ** 2) + eps) * weight              (from the unrounded h)
    scale = max(max|y| / 448, 1e-12);  codes = e4m3(y / scale)

bf16 and fp16; the kernels are in ``csrc/qik_norm.cu``, the argument checks in ``csrc/calls.cpp``.
"""
from __future__ import annotations

import torch

from . import _calls


def fused_add_rms_norm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor,
                       eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """x, residual: [..., N] bf16 or fp16 (residual None: the plain norm of x), N a multiple of 8
    up to 32768; weight [N] of the same type or fp32.  Returns (norm, x + residual), both
    contiguous in x's type; the second is x itself without a residual."""
    return _calls.add_rms_norm(x, residual, weight, eps, None)


def fused_add_rms_norm_e4m3(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float,
                            scales: str = "tensor") -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """As ``fused_add_rms_norm`` with the norm quantized: returns (codes e4m3 [..., N],
    scale fp32, x + residual).  ``scales="tensor"``: one scale, shape [1], which
    ``FP8Linear.forward_e4m3`` takes; ``scales="row"``: one for each row, shape [...] (the linears
    of this library take one scale only and refuse them).  NaN in the norm reaches its scale."""
    return _calls.add_rms_norm(x, residual, weight, eps, scales or "")
