"""Attention of new tokens over a paged KV cache (``qik.paged_kv``), next to the block-causal
attention over a contiguous slab of ``qik.triton_attention``.

One call serves a batch of sequences that each bring one token (decoding), a few (drafts),
a chunk or a whole prompt; query heads may share key heads; rows see the cache causally, or
all of it, or the last ``window`` keys and the first ``sinks``.  The kernels
(``csrc/qik_paged_attn.cu``) read the lengths on the device, so a captured graph follows them.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib as L
from .rotary import check_pages

_TYPES = (torch.bfloat16, torch.float16)


def paged_attention(
    q: torch.Tensor,             # [T, HQ, D] new tokens of all sequences, one after another
    k_pages: torch.Tensor,       # [pages, HK, page, D]
    v_pages: torch.Tensor,
    page_table: torch.Tensor,    # [B, W] int32
    seq_lens: torch.Tensor,      # [B] int32: tokens in the cache, the new ones among them
    query_starts: torch.Tensor,  # [B + 1] int32: sequence i's rows of q
    max_new: int,                # most new tokens of a sequence
    max_kv: int | None = None,   # most tokens of a sequence (None: what the page table can hold)
    sm_scale: float | None = None,
    causal: bool = True,
    window: int = 0,
    sinks: int = 0,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """softmax(q . k * sm_scale) . v of each new token over its sequence's keys, [T, HQ, D].

    The new tokens are the last of their sequence, already stored.  Row j of n in a sequence of
    ``kv`` tokens sees the keys t <= kv - n + j (``causal``) or all kv; with ``window`` (causal
    only) those with t > kv - n + j - window or t < ``sinks``.  A row that sees nothing is 0.
    Places that no row of a sequence sees may hold anything, NaN included.  ``sm_scale`` is
    D ** -0.5 by default.  ``out`` ([T, HQ, D], unit column stride) receives the result; rows
    behind query_starts[B] are not written.  No sequence may bring more than ``max_new``
    tokens; ``max_kv`` only chooses launch shapes.  Lengths, starts and page numbers outside
    their tensors are skipped and set ``STATUS_BAD_INDEX`` (``qik._lib.device_status``)."""
    dev = q.device
    if not q.is_cuda:
        raise ValueError("qik: q must be a CUDA tensor (the kernels have no CPU path)")
    if q.dtype not in _TYPES:
        raise TypeError(f"qik: paged_attention: bf16 or fp16, got {q.dtype}")
    if q.dim() != 3 or q.shape[2] not in (64, 128):
        raise ValueError(f"qik: q is {tuple(q.shape)}: expected [tokens, heads, 64 or 128]")
    T, HQ, D = q.shape
    check_pages(k_pages, v_pages, q)
    pages, HK, page, _ = k_pages.shape
    if HQ == 0 or HQ % HK:
        raise ValueError(f"qik: {HQ} query heads do not share {HK} key heads evenly")
    B = seq_lens.shape[0]
    for name, t, dim in (("page_table", page_table, 2), ("seq_lens", seq_lens, 1), ("query_starts", query_starts, 1)):
        if t.dtype != torch.int32 or t.device != dev or t.dim() != dim:
            raise ValueError(f"qik: {name} is {tuple(t.shape)} {t.dtype} on {t.device}: expected int32 on {dev}")
    if page_table.shape[0] != B or query_starts.shape[0] != B + 1:
        raise ValueError(f"qik: page_table {tuple(page_table.shape)}, seq_lens {tuple(seq_lens.shape)} and query_starts "
                         f"{tuple(query_starts.shape)} are not of one batch")
    W = page_table.shape[1]
    if not 0 <= max_new <= T:
        raise ValueError(f"qik: max_new is {max_new}, q has {T} tokens")
    if max_kv is None:
        max_kv = W * page
    if window < 0 or sinks < 0 or max_kv < 0 or (window and not causal):
        raise ValueError(f"qik: window {window}, sinks {sinks}, max_kv {max_kv}, causal {causal} (a window needs causal)")
    if sm_scale is None:
        sm_scale = D ** -0.5
    elif not 0.0 < sm_scale < 1e30:
        raise ValueError(f"qik: sm_scale must be positive and finite, got {sm_scale}")
    st, sh, sd = q.stride()
    if sd != 1 or st % 8 or sh % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        st, sh, _ = q.stride()
    if out is None:
        out = torch.empty((T, HQ, D), dtype=q.dtype, device=dev)
        o_st, o_sh = HQ * D, D
    else:
        if out.shape != q.shape or out.dtype != q.dtype or out.device != dev:
            raise ValueError(f"qik: out is {tuple(out.shape)} {out.dtype} on {out.device}: expected {tuple(q.shape)} {q.dtype}")
        o_st, o_sh, sd = out.stride()
        if sd != 1 or o_st % 8 or o_sh % 8 or out.data_ptr() % 16:
            raise ValueError("qik: out needs a unit column stride, strides of 16 bytes and 16-byte alignment")
    if page_table.stride(1) != 1 and W > 1:
        page_table = page_table.contiguous()
    if not seq_lens.is_contiguous():
        seq_lens = seq_lens.contiguous()
    if not query_starts.is_contiguous():
        query_starts = query_starts.contiguous()
    k0, kh, ks, _ = k_pages.stride()
    v0, vh, vs, _ = v_pages.stride()
    a = L.PagedAttnArgs(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(), page_table.data_ptr(),
                        seq_lens.data_ptr(), query_starts.data_ptr(), B, T, HQ, HK, D, W, pages, page, max_new, max_kv,
                        st, sh, o_st, o_sh, page_table.stride(0), k0, kh, ks, v0, vh, vs, sm_scale, window, sinks,
                        (L.PAGED_CAUSAL if causal else 0) | (L.PAGED_F16 if q.dtype == torch.float16 else 0))
    ref = ctypes.byref(a)
    # the workspace is the caller's stream's: torch hands its memory on only to later work there
    with_ws = L.on_device("qik_paged_attention_workspace_bytes", dev, ref)
    ws = torch.empty(with_ws, dtype=torch.uint8, device=dev) if with_ws else None
    L.launch("qik_paged_attention", dev, ref, None if ws is None else ws.data_ptr(), with_ws,
             L.status_word(dev).data_ptr())
    return out
