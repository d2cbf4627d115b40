"""Rotary positions for a transformer decoder, next to ``fused_rms_norm_rope`` of
``qik.triton_fused`` (which turns whole heads by complex interleaved frequencies after an
RMS norm; the reference has no other form).

``rotary_table`` makes the cosines and sines once, from angles in 64 bits, with the usual
scalings for long contexts; ``apply_rotary`` turns q and k by them, in interleaved pairs or
in halves, over the whole head or its first columns; ``rotary_store`` does that and stores
the turned k and v in the pages of a cache (``qik.paged_kv``) in the same kernel
(``csrc/qik_rotary.cu``).
"""
from __future__ import annotations

import math

import torch

from . import _calls

SCALINGS = ("none", "linear", "ntk", "yarn", "bands")


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       original_positions: int = 4096, fast_turns: float | None = None,
                       slow_turns: float = 1.0) -> tuple[torch.Tensor, float]:
    """Radians per position of each of the rotary_dim / 2 pairs (64 bits, on the host) and
    the factor on the cosines and sines.  With f_i = base ** (-2 i / rotary_dim):

    * ``none``   f_i;
    * ``linear`` f_i / factor (positions interpolated);
    * ``ntk``    base * factor ** (rotary_dim / (rotary_dim - 2)) in base's place: the fastest
      pair keeps its frequency, the slowest is divided by factor;
    * ``yarn``   between f_i (pairs that turn over ``fast_turns`` = 32 times in
      ``original_positions``) and f_i / factor (under ``slow_turns`` = 1 times), by a ramp over
      the pair's index; the table is scaled by 0.1 ln(factor) + 1;
    * ``bands``  the same ends with ``fast_turns`` = 4, by a ramp over the number of turns.
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"qik: rotary_dim must be even, got {rotary_dim}")
    if scaling not in SCALINGS:
        raise ValueError(f"qik: scaling is one of {SCALINGS}, got {scaling!r}")
    if not (base > 1.0 and factor > 0.0 and original_positions > 0):
        raise ValueError(f"qik: base {base}, factor {factor}, original_positions {original_positions}")
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / rotary_dim)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "ntk":
        if rotary_dim == 2:
            return f, 1.0
        return (base * factor ** (rotary_dim / (rotary_dim - 2))) ** (-2.0 * i / rotary_dim), 1.0
    if scaling == "yarn":
        def pair_of(turns: float) -> float:
            return rotary_dim * math.log(original_positions / (turns * 2 * math.pi)) / (2 * math.log(base))
        low = max(0, math.floor(pair_of(32.0 if fast_turns is None else fast_turns)))
        high = min(rotary_dim - 1, math.ceil(pair_of(slow_turns)))
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    if scaling == "bands":
        fast = 4.0 if fast_turns is None else fast_turns
        mix = ((original_positions * f / (2 * math.pi) - slow_turns) / (fast - slow_turns)).clamp(0, 1)
        return f / factor * (1 - mix) + f * mix, 1.0
    return f, 1.0


def rotary_table(rotary_dim: int, max_positions: int, *, device: torch.device | str = "cuda",
                 **scaling) -> tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin), fp32 [max_positions, rotary_dim / 2] on ``device``; keyword arguments as
    ``rotary_frequencies``.  Angles are formed and reduced in 64 bits."""
    if max_positions <= 0:
        raise ValueError(f"qik: max_positions must be positive, got {max_positions}")
    f, gain = rotary_frequencies(rotary_dim, **scaling)
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * f.to(device)
    return (angle.cos() * gain).float(), (angle.sin() * gain).float()


def apply_rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: tuple[torch.Tensor, torch.Tensor],
                 interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """q [T, HQ, D], k [T, HK, D] (bf16 or fp16, D 64, 128 or 256, any strides with a unit column
    stride: views of a fused projection are read in place); positions [T] int32 or int64;
    table from ``rotary_table``, for a multiple of 16 columns.  Returns the turned q and k,
    contiguous.  A position outside the table gives zeros and ``STATUS_BAD_INDEX`` in the
    device's status word (``qik._lib.device_status``)."""
    return _calls.rotary(q, k, None, positions, *table, None, None, None, interleaved)


def rotary_store(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                 table: tuple[torch.Tensor, torch.Tensor], slots: torch.Tensor, k_pages: torch.Tensor,
                 v_pages: torch.Tensor, interleaved: bool = False) -> torch.Tensor:
    """``apply_rotary`` whose k goes, with v [T, HK, D], into one layer's pages [pages, HK,
    page, D] (page a power of two from 16 to 4096): token t at page slots[t] // page, place
    slots[t] % page.  slots [T] int32 or int64, distinct; a negative slot stores nothing
    (padding), one behind the last page stores nothing and sets ``STATUS_BAD_INDEX``, and so does
    a token whose position is outside the table.  Returns the turned q."""
    return _calls.rotary(q, k, v, positions, *table, slots, k_pages, v_pages, interleaved)
