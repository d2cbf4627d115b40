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


def _heads(t: torch.Tensor, name: str, T: int, D: int, dtype: torch.dtype, dev: torch.device) -> tuple:
    """t as [T, H, D] with a unit column stride, 16-byte rows and heads (copied otherwise), and
    its heads, token and head strides."""
    s = t.shape
    if len(s) != 3 or s[0] != T or s[2] != D or t.dtype != dtype or t.device != dev:
        raise ValueError(f"qik: {name} is {tuple(s)} {t.dtype} on {t.device}: expected [{T}, heads, {D}] {dtype} on {dev}")
    st, sh, sd = t.stride()
    if sd != 1 or (st | sh) % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        st, sh, sd = t.stride()
    return t, s[1], st, sh


def _index(t: torch.Tensor, name: str, T: int, dev: torch.device) -> torch.Tensor:
    if t.shape != (T,) or t.dtype not in _INTS or t.device != dev:
        raise ValueError(f"qik: {name} is {tuple(t.shape)} {t.dtype} on {t.device}: expected [{T}] int32 or int64 on {dev}")
    return t if t.is_contiguous() else t.contiguous()


def _run(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor | None, positions: torch.Tensor, table: tuple,
         slots: torch.Tensor | None, k_out: torch.Tensor | None, v_out: torch.Tensor | None, interleaved: bool) -> tuple:
    if not q.is_cuda:
        raise ValueError("qik: q must be a CUDA tensor (the kernels have no CPU path)")
    dtype, dev = q.dtype, q.device
    if dtype not in _FLOATS:
        raise TypeError(f"qik: rotary: bf16 or fp16, got {dtype}")
    if q.dim() != 3 or q.shape[2] not in (64, 128, 256):
        raise ValueError(f"qik: q is {tuple(q.shape)}: expected [tokens, heads, 64, 128 or 256]")
    T, HQ, D = q.shape
    cos, sin = table
    P, pairs = cos.shape if cos.dim() == 2 else (0, 0)
    if cos.dtype != torch.float32 or sin.dtype != torch.float32 or sin.shape != cos.shape or P == 0 or \
            not (cos.is_contiguous() and sin.is_contiguous()) or cos.device != dev or sin.device != dev:
        raise ValueError("qik: table is (cos, sin), contiguous fp32 [positions, rotary_dim / 2] on q's device")
    if pairs == 0 or pairs % 8 or 2 * pairs > D:
        raise ValueError(f"qik: a table for {2 * pairs} columns does not fit heads of {D} (a multiple of 16)")
    q, _, q_st, q_sh = _heads(q, "q", T, D, dtype, dev)
    k, HK, k_st, k_sh = _heads(k, "k", T, D, dtype, dev)
    positions = _index(positions, "positions", T, dev)
    flags = ((L.ROTARY_INTERLEAVED if interleaved else 0) | (L.ROTARY_F16 if dtype == torch.float16 else 0)
             | (L.ROTARY_POS64 if positions.dtype == torch.int64 else 0))
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if slots is None:
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        v_ptr = v_out_ptr = slots_ptr = 0
        v_st = v_sh = page = pages = 0
        strides = (0, 0, 0, 0, 0, 0)
    else:
        v, HV, v_st, v_sh = _heads(v, "v", T, D, dtype, dev)
        if HV != HK:
            raise ValueError(f"qik: v has {HV} heads, k {HK}")
        slots = _index(slots, "slots", T, dev)
        pages, heads, page, strides = check_pages(k_out, v_out, D, dtype, dev)
        if heads != HK:
            raise ValueError(f"qik: pages hold {heads} heads, k has {HK}")
        flags |= L.ROTARY_PAGED | (L.ROTARY_SLOT64 if slots.dtype == torch.int64 else 0)
        v_ptr, v_out_ptr, slots_ptr = v.data_ptr(), v_out.data_ptr(), slots.data_ptr()
    idx = dev.index
    if T:
        L.launch("qik_rotary", idx,
                 L.pack_rotary(q.data_ptr(), k.data_ptr(), v_ptr, q_out.data_ptr(), k_out.data_ptr(), v_out_ptr,
                               positions.data_ptr(), slots_ptr, cos.data_ptr(), sin.data_ptr(), T, HQ, HK, D, 2 * pairs, P,
                               q_st, q_sh, k_st, k_sh, v_st, v_sh, page, pages, *strides, flags), L.status_ptr(idx))
    return q_out, k_out


def apply_rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, table: tuple[torch.Tensor, torch.Tensor],
                 interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """q [T, HQ, D], k [T, HK, D] (bf16 or fp16, any strides with a unit column stride: views of
    a fused projection are read in place); positions [T] int32 or int64; table from
    ``rotary_table``.  Returns the turned q and k, contiguous.  A position outside the
    table gives zeros and ``STATUS_BAD_INDEX`` in the device's status word."""
    return _run(q, k, None, positions, table, None, None, None, interleaved)


def rotary_store(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                 table: tuple[torch.Tensor, torch.Tensor], slots: torch.Tensor, k_pages: torch.Tensor,
                 v_pages: torch.Tensor, interleaved: bool = False) -> torch.Tensor:
    """``apply_rotary`` whose k goes, with v [T, HK, D], into one layer's pages [pages, HK,
    page, D] (page a power of two): token t at page slots[t] // page, place slots[t] % page.
    slots [T] int32 or int64, distinct; a negative slot stores nothing (padding), one behind the
    last page stores nothing and sets ``STATUS_BAD_INDEX``.  Returns the turned q."""
    return _run(q, k, v, positions, table, slots, k_pages, v_pages, interleaved)[0]


def check_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, D: int, dtype: torch.dtype, dev: torch.device) -> tuple:
    """One layer's page pools: [pages, heads, page, D], page a power of two of 16 to 4096 tokens,
    unit column stride, 16-byte strides.  Returns pages, heads, page and the page, head and token
    strides of both."""
    s = k_pages.shape
    if len(s) != 4 or v_pages.shape != s or s[3] != D or k_pages.dtype != dtype or v_pages.dtype != dtype or \
            k_pages.device != dev or v_pages.device != dev:
        raise ValueError(f"qik: pages {tuple(s)} {k_pages.dtype} on {k_pages.device} and {tuple(v_pages.shape)} "
                         f"{v_pages.dtype} on {v_pages.device}: expected two [pages, heads, page, {D}] {dtype} on {dev}")
    pages, heads, page, _ = s
    if pages == 0 or heads == 0 or page < 16 or page > 4096 or page & (page - 1):
        raise ValueError(f"qik: pages {tuple(s)}: a page is a power of two of 16 to 4096 tokens")
    a, b, c, d = k_pages.stride()
    e, f, g, h = v_pages.stride()
    if d != 1 or h != 1 or (a | b | c | e | f | g) % 8 or (k_pages.data_ptr() | v_pages.data_ptr()) % 16:
        raise ValueError("qik: pages need a unit column stride, strides of 16 bytes and 16-byte alignment")
    return pages, heads, page, (a, b, c, e, f, g)
