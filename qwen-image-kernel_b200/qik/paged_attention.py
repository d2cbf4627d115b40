"""Attention of new tokens over a paged KV cache (``qik.paged_kv``), next to the block-causal
attention over a contiguous slab of ``qik.triton_attention``.

One call serves a batch of sequences that each bring one token (decoding), a few (drafts),
a chunk or a whole prompt; query heads may share key heads; rows see the cache causally, or
all of it, or the last ``window`` keys and the first ``sinks``.  The kernels
(``csrc/qik_paged_attn.cu``) read the lengths on the device, so a captured graph follows them.
"""
from __future__ import annotations

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
    if not q.is_cuda:
        raise ValueError("qik: q must be a CUDA tensor (the kernels have no CPU path)")
    dev, dtype = q.device, q.dtype
    if dtype not in _TYPES:
        raise TypeError(f"qik: paged_attention: bf16 or fp16, got {dtype}")
    if q.dim() != 3 or q.shape[2] not in (64, 128):
        raise ValueError(f"qik: q is {tuple(q.shape)}: expected [tokens, heads, 64 or 128]")
    T, HQ, D = q.shape
    pages, HK, page, strides = check_pages(k_pages, v_pages, D, dtype, dev)
    if HQ == 0 or HQ % HK:
        raise ValueError(f"qik: {HQ} query heads do not share {HK} key heads evenly")
    i32 = torch.int32
    if page_table.dtype != i32 or seq_lens.dtype != i32 or query_starts.dtype != i32 or page_table.device != dev or \
            seq_lens.device != dev or query_starts.device != dev:
        raise ValueError(f"qik: page_table, seq_lens and query_starts must be int32 on {dev}")
    if page_table.dim() != 2 or seq_lens.dim() != 1 or query_starts.dim() != 1 or \
            page_table.shape[0] != seq_lens.shape[0] or query_starts.shape[0] != seq_lens.shape[0] + 1:
        raise ValueError(f"qik: page_table {tuple(page_table.shape)}, seq_lens {tuple(seq_lens.shape)} and query_starts "
                         f"{tuple(query_starts.shape)}: expected [B, W], [B] and [B + 1]")
    B, W = page_table.shape
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
    q_st, q_sh, sd = q.stride()
    if sd != 1 or (q_st | q_sh) % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        q_st, q_sh, _ = q.stride()
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != dtype or out.device != dev:
        raise ValueError(f"qik: out is {tuple(out.shape)} {out.dtype} on {out.device}: expected {tuple(q.shape)} {dtype}")
    o_st, o_sh, sd = out.stride()
    if sd != 1 or (o_st | o_sh) % 8 or out.data_ptr() % 16:
        raise ValueError("qik: out needs a unit column stride, strides of 16 bytes and 16-byte alignment")
    t_st, td = page_table.stride()
    if td != 1 and W > 1:
        page_table = page_table.contiguous()
        t_st = W
    if not seq_lens.is_contiguous():
        seq_lens = seq_lens.contiguous()
    if not query_starts.is_contiguous():
        query_starts = query_starts.contiguous()
    args = L.pack_paged_attn(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(), page_table.data_ptr(),
                             seq_lens.data_ptr(), query_starts.data_ptr(), B, T, HQ, HK, D, W, pages, page, max_new, max_kv,
                             q_st, q_sh, o_st, o_sh, t_st, *strides, sm_scale, window, sinks,
                             (L.PAGED_CAUSAL if causal else 0) | (L.PAGED_F16 if dtype == torch.float16 else 0))
    idx = dev.index
    # a workspace of this call alone: torch hands its memory on only to later work of the stream
    n = L.on_device("qik_paged_attention_workspace_bytes", idx, args)
    ws = q.new_empty(n, dtype=torch.uint8) if n else None
    L.launch("qik_paged_attention", idx, args, None if ws is None else ws.data_ptr(), n, L.status_ptr(idx))
    return out
