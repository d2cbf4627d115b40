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

import ctypes
import math

import torch

from . import _lib as L

SCALINGS = ("none", "linear", "ntk", "yarn", "bands")
_FLOATS = (torch.bfloat16, torch.float16)
_INTS = (torch.int32, torch.int64)


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


def _heads(t: torch.Tensor, name: str, like: torch.Tensor) -> torch.Tensor:
    """t as [T, H, D] with a unit column stride, 16-byte rows and heads (copied otherwise)."""
    if t.dim() != 3 or t.dtype != like.dtype or t.device != like.device or t.shape[0] != like.shape[0] or \
            t.shape[2] != like.shape[2]:
        raise ValueError(f"qik: {name} is {tuple(t.shape)} {t.dtype} on {t.device}: expected [{like.shape[0]}, heads, "
                         f"{like.shape[2]}] {like.dtype} on {like.device}")
    st, sh, sd = t.stride()
    if sd != 1 or st % 8 or sh % 8 or t.data_ptr() % 16:
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _index(t: torch.Tensor, name: str, like: torch.Tensor) -> torch.Tensor:
    if t.dtype not in _INTS or t.device != like.device or t.dim() != 1 or t.shape[0] != like.shape[0]:
        raise ValueError(f"qik: {name} is {tuple(t.shape)} {t.dtype} on {t.device}: expected [{like.shape[0]}] int32 or "
                         f"int64 on {like.device}")
    return t if t.is_contiguous() else t.contiguous()


def _args(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: tuple, interleaved: bool) -> tuple:
    if not q.is_cuda:
        raise ValueError("qik: q must be a CUDA tensor (the kernels have no CPU path)")
    if q.dtype not in _FLOATS:
        raise TypeError(f"qik: rotary: bf16 or fp16, got {q.dtype}")
    if q.dim() != 3 or q.shape[2] not in (64, 128, 256):
        raise ValueError(f"qik: q is {tuple(q.shape)}: expected [tokens, heads, 64, 128 or 256]")
    cos, sin = table
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or cos.shape != sin.shape or cos.dim() != 2 or \
            not (cos.is_contiguous() and sin.is_contiguous()) or cos.device != q.device or sin.device != q.device:
        raise ValueError("qik: table is (cos, sin), contiguous fp32 [positions, rotary_dim / 2] on q's device")
    rot = 2 * cos.shape[1]
    if rot % 16 or not 0 < rot <= q.shape[2] or cos.shape[0] == 0:
        raise ValueError(f"qik: a table for {rot} columns does not fit heads of {q.shape[2]} (a multiple of 16)")
    q, k, positions = _heads(q, "q", q), _heads(k, "k", q), _index(positions, "positions", q)
    a = L.RotaryArgs()
    a.q, a.k, a.positions, a.cos, a.sin = (q.data_ptr(), k.data_ptr(), positions.data_ptr(), cos.data_ptr(),
                                           sin.data_ptr())
    a.T, a.HQ, a.D = q.shape
    a.HK, a.rot, a.P = k.shape[1], rot, cos.shape[0]
    a.q_st, a.q_sh, _ = q.stride()
    a.k_st, a.k_sh, _ = k.stride()
    a.flags = ((L.ROTARY_INTERLEAVED if interleaved else 0) | (L.ROTARY_F16 if q.dtype == torch.float16 else 0)
               | (L.ROTARY_POS64 if positions.dtype == torch.int64 else 0))
    return a, q, k, positions


def apply_rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: tuple[torch.Tensor, torch.Tensor],
                 interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """q [T, HQ, D], k [T, HK, D] (bf16 or fp16, any strides with a unit column stride: views of
    a fused projection are read in place); positions [T] int32 or int64; table from
    ``rotary_table``.  Returns the turned q and k, contiguous.  A position outside the
    table gives zeros and ``STATUS_BAD_INDEX`` in the device's status word."""
    a, q, k, positions = _args(q, k, positions, table, interleaved)
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    a.q_out, a.k_out = q_out.data_ptr(), k_out.data_ptr()
    L.launch("qik_rotary", q.device, ctypes.byref(a), L.status_word(q.device).data_ptr())
    return q_out, k_out


def rotary_store(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                 table: tuple[torch.Tensor, torch.Tensor], slots: torch.Tensor, k_pages: torch.Tensor,
                 v_pages: torch.Tensor, interleaved: bool = False) -> torch.Tensor:
    """``apply_rotary`` whose k goes, with v [T, HK, D], into one layer's pages [pages, HK,
    page, D] (page a power of two): token t at page slots[t] // page, place slots[t] % page.
    slots [T] int32 or int64, distinct; a negative slot stores nothing (padding), one behind the
    last page stores nothing and sets ``STATUS_BAD_INDEX``.  Returns the turned q."""
    a, q, k, positions = _args(q, k, positions, table, interleaved)
    v, slots = _heads(v, "v", q), _index(slots, "slots", q)
    if v.shape != k.shape:
        raise ValueError(f"qik: v is {tuple(v.shape)}, k {tuple(k.shape)}")
    check_pages(k_pages, v_pages, q, k.shape[1])
    pages, _, page, _ = k_pages.shape
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    a.q_out, a.k_out, a.v_out, a.v, a.slots = (q_out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), v.data_ptr(),
                                               slots.data_ptr())
    a.v_st, a.v_sh, _ = v.stride()
    a.page, a.pages = page, pages
    a.kp_s0, a.kp_sh, a.kp_ss, _ = k_pages.stride()
    a.vp_s0, a.vp_sh, a.vp_ss, _ = v_pages.stride()
    a.flags |= L.ROTARY_PAGED | (L.ROTARY_SLOT64 if slots.dtype == torch.int64 else 0)
    L.launch("qik_rotary", q.device, ctypes.byref(a), L.status_word(q.device).data_ptr())
    return q_out


def check_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, like: torch.Tensor, heads: int | None = None) -> None:
    """One layer's page pools: [pages, heads, page, D] of like's type and device, page a power of
    two of at least 16 tokens, unit column stride and 16-byte strides."""
    s = k_pages.shape
    if v_pages.shape != s or len(s) != 4 or k_pages.dtype != like.dtype or v_pages.dtype != like.dtype or \
            k_pages.device != like.device or v_pages.device != like.device or s[3] != like.shape[-1]:
        raise ValueError(f"qik: pages {tuple(s)} {k_pages.dtype} and {tuple(v_pages.shape)} {v_pages.dtype}: expected two "
                         f"[pages, heads, page, {like.shape[-1]}] {like.dtype} on {like.device}")
    if heads is not None and s[1] != heads:
        raise ValueError(f"qik: pages hold {s[1]} heads, k has {heads}")
    if s[0] == 0 or s[1] == 0 or s[2] < 16 or s[2] > 4096 or s[2] & (s[2] - 1):
        raise ValueError(f"qik: pages {tuple(s)}: a page is a power of two of 16 to 4096 tokens")
    for t in (k_pages, v_pages):
        a, b, c, d = t.stride()
        if d != 1 or a % 8 or b % 8 or c % 8 or min(a, b, c) < 0 or t.data_ptr() % 16:
            raise ValueError("qik: pages need a unit column stride, strides of 16 bytes and 16-byte alignment")
